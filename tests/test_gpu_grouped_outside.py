"""A position whose row lies outside x gets zeros, whatever the bank and its
scales hold, in each of grouped_matmul's kernels."""
from __future__ import annotations

import pytest
import torch

import vxmoe

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("P,E,N,K", [(1, 1, 40, 64), (6, 2, 33, 64), (50, 1, 3, 528), (300, 3, 96, 128),
                                     (300, 2, 131, 1040), (1000, 1, 256, 1040), (500, 40, 260, 1040)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_outside_get_zeros_from_any_bank(kind, P, E, N, K, bad):
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn((37, K), device="cuda", generator=g).bfloat16()
    w = torch.randn((E, N, K), device="cuda", generator=g).bfloat16()
    offsets = torch.tensor([P * e // E for e in range(E + 1)], device="cuda", dtype=torch.int32)
    rows = torch.randint(0, 37 * 2, (P,), device="cuda", generator=g, dtype=torch.int32)
    outside = torch.rand(P, device="cuda", generator=g) < 0.3
    outside[P // 2] = True
    values = torch.tensor([-1, 74, 75, 2 ** 31 - 1, -2 ** 31], device="cuda", dtype=torch.int32)
    rows[outside] = values[torch.arange(int(outside.sum()), device="cuda") % 5]
    xs = ws = None
    if kind == "e4m3":
        x, w = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
        xs, ws = torch.rand(37, device="cuda") + 0.5, torch.rand((E, N), device="cuda") + 0.5
    kw = dict(rows=rows, slots=2, x_scales=xs, w_scales=ws)
    clean = vxmoe.grouped_matmul(x, w, offsets, **kw)
    assert not clean[outside].float().any() and clean[~outside].float().isfinite().all()
    # one output's scale, or one input of one output of every expert
    ws2, w2 = ws, w.float()
    w2[:, N // 2, K // 3] = bad if kind == "bf16" else float("nan")
    w2 = w2.to(w.dtype)
    if kind == "e4m3":
        ws2 = ws.clone()
        ws2[:, 0] = bad
    got = vxmoe.grouped_matmul(x, w2, offsets, rows=rows, slots=2, x_scales=xs, w_scales=ws2)
    assert not got[outside].float().any(), "a padded position took something from the bank"
    assert not got[~outside][:, N // 2].float().isfinite().any()
    keep = [n for n in range(N) if n != N // 2 and not (kind == "e4m3" and n == 0)]
    assert torch.equal(got[:, keep].view(torch.int16), clean[:, keep].view(torch.int16))
