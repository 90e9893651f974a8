"""lora_add's inner values at the end of the float32 range."""
from __future__ import annotations

import pytest
import torch

import vxmoe
from rows64 import BF16, lora64, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 40, 300])
def test_inner_values_between_the_largest_bf16_and_the_largest_float32(T):
    """h = 3.4e38 is finite in float32 and rounds to infinity in bf16; B brings it back."""
    K, N, L, R = 64, 40, 3, 16
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.zeros((T, K), device="cuda", dtype=torch.bfloat16)
    x[:, 5] = 1.0
    x[1::2, 5] = -1.0
    a = torch.zeros((L, R, K), device="cuda", dtype=torch.bfloat16)
    a[:, :, 5] = 1.0
    b = (torch.rand((L, N, R), device="cuda", generator=g) * 2.0 ** -100).bfloat16()
    y = torch.randn((T, N), device="cuda", generator=g).bfloat16()
    scales = torch.tensor([3.4e38, 3.3897e38, -torch.finfo(torch.float32).max], device="cuda")
    ids = torch.arange(T, device="cuda", dtype=torch.int32) % 4      # one in four without an adapter
    got = vxmoe.lora_add(y, x, a, b, ids, scales=scales)
    want, tol = lora64(y, x, a, b, ids, scales=scales)
    within(got, want, want.abs() * BF16 + tol * (1 + BF16), f"T={T}")
    # no finite value comes from one that is none
    got = vxmoe.lora_add(y, x * float("inf"), a, b, ids, scales=scales)
    assert not got[ids < 3].float().isfinite().any() and torch.equal(got[ids == 3], y[ids == 3])
