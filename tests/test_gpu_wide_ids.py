"""Ids of more than 32 bits name no row, no adapter and no position: they are
not cut down to ones that do."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import vxmoe

pytestmark = pytest.mark.gpu


def normal(*shape, seed=1):
    return torch.randn(shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).bfloat16()


@pytest.mark.parametrize("T", [6, 300])
def test_adapters_beyond_32_bits(T):
    y, x, a, b = normal(T, 40), normal(T, 64, seed=2), normal(2, 8, 64, seed=3), normal(2, 40, 8, seed=4)
    ids = (torch.arange(T) % 6).long()
    far = torch.tensor([0, 2 ** 32, 2 ** 32 + 1, 1, -2 ** 32, 2 ** 63 - 1])[ids]
    near = torch.tensor([0, -1, -1, 1, -1, -1])[ids]
    want = vxmoe.lora_add(y, x, a, b, near.int().cuda())
    for given in (far, far.cuda(), far.numpy(), far.tolist()):
        assert torch.equal(vxmoe.lora_add(y, x, a, b, given), want)
    unsigned = torch.tensor([0, 2 ** 31, 2 ** 32 - 1, 1, 7, 9])[ids].numpy().astype(np.uint32)
    assert torch.equal(vxmoe.lora_add(y, x, a, b, unsigned), want)
    assert torch.equal(vxmoe.lora_add(y, x, a, b, torch.from_numpy(unsigned).cuda()), want)
    small = torch.tensor([0, 200, 255, 1, 7, 9])[ids].numpy()
    for kind in (np.uint8, np.int16, np.uint64):
        assert torch.equal(vxmoe.lora_add(y, x, a, b, small.astype(kind)), want)


@pytest.mark.parametrize("P", [6, 300])
def test_rows_and_offsets_beyond_32_bits(P):
    x, w = normal(4, 64), normal(2, 24, 64, seed=2)
    offsets = torch.tensor([0, P // 2, P], dtype=torch.int32, device="cuda")
    at = torch.arange(P) % 4
    near, far = torch.tensor([0, -1, 3, -1])[at], torch.tensor([0, 2 ** 32 + 1, 3, -2 ** 33])[at]
    want = vxmoe.grouped_matmul(x, w, offsets, rows=near.int().cuda())
    assert not want[at.cuda() % 2 == 1].float().any() and want[0].float().any()
    assert torch.equal(vxmoe.grouped_matmul(x, w, offsets, rows=far), want)
    assert torch.equal(vxmoe.grouped_matmul(x, w, offsets, rows=far.cuda()), want)
    far = torch.tensor([-2 ** 40, P // 2, 2 ** 40])      # clamped to [0, P]
    assert torch.equal(vxmoe.grouped_matmul(x, w, far, rows=near), want)
    far = torch.tensor([0, P // 2, 2 ** 32 - 5], dtype=torch.int64).numpy().astype(np.uint32)
    assert torch.equal(vxmoe.grouped_matmul(x, w, far, rows=near), want)
