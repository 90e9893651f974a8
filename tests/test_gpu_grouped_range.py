"""grouped_matmul's scales at the ends of the float32 range, in each of its
kernels: the product of a row's and an output's scale alone leaves the range,
the value does not."""
from __future__ import annotations

import pytest
import torch

import vxmoe
from rows64 import BF16, F32, grouped64, sum_tol, within

pytestmark = pytest.mark.gpu

# few rows; positions as M; CTA pairs (by the positions, the experts and the length of the rows)
SHAPES = [(5, 2, 96, 512), (300, 3, 96, 512), (300, 2, 130, 1024)]


def operands(P, E, N, K):
    g = torch.Generator("cuda").manual_seed(1)

    def values(*shape):   # of one sign, so that sums reach 2^25
        return (torch.rand(shape, device="cuda", generator=g) * 200 + 200).to(torch.float8_e4m3fn)
    offsets = torch.tensor([0] + [P * (e + 1) // E for e in range(E)], device="cuda", dtype=torch.int32)
    return values(P, K), values(E, N, K), offsets, torch.rand(P, device="cuda", generator=g) + 0.5, \
        torch.rand((E, N), device="cuda", generator=g) + 0.5


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("P,E,N,K", SHAPES)
@pytest.mark.parametrize("px,pw", [(-75, -70), (-75, -73), (-126, -22), (-20, -126), (-70, -60), (-140, 20), (15, -139),
                                   (100, -120), (-120, 100), (110, -140)])
def test_scales_whose_product_leaves_the_range(px, pw, P, E, N, K, gather):
    x, w, offsets, xs, ws = operands(P, E, N, K)
    xs, ws = xs * 2.0 ** px, ws * 2.0 ** pw
    xs[::3] = -xs[::3]
    xs[1] = 0
    ws[0, 2] = 0
    rows = torch.randint(0, P, (P,), device="cuda", dtype=torch.int32,
                         generator=torch.Generator("cuda").manual_seed(2)) if gather else None
    got = vxmoe.grouped_matmul(x, w, offsets, rows=rows, x_scales=xs, w_scales=ws)
    want, size = grouped64(x, w, offsets, rows, 1, xs, ws)
    # bf16's step below its normal range is 2^-133, float32's 2^-149
    within(got, want, want.abs() * (BF16 + 8 * F32) + size * sum_tol(K) + 2.0 ** -134 + 2.0 ** -148, f"{px} {pw}")


@pytest.mark.parametrize("P,E,N,K", SHAPES)
def test_small_sums_under_scales_whose_product_overflows(P, E, N, K):
    """One input of 2^-9 times another of 2^-9, scales of 2^70 and 2^66: 2^118."""
    x, w, offsets, xs, ws = operands(P, E, N, K)
    x, w = x.float().zero_(), w.float().zero_()
    x[:, 7] = 2.0 ** -9
    w[:, :, 7] = 2.0 ** -9
    x, w = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
    xs, ws = xs * 2.0 ** 70, ws * 2.0 ** 66
    got = vxmoe.grouped_matmul(x, w, offsets, x_scales=xs, w_scales=ws)
    want, _ = grouped64(x, w, offsets, None, 1, xs, ws)
    within(got, want, want.abs() * (BF16 + 8 * F32), "large scales")
