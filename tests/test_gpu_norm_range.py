"""add_rms_norm on rows whose squares leave the float32 range, at both of its
ends, in every row variant (one warp, one CTA, rows read twice, narrow
accesses), against the definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

import vxmoe
from rows64 import BF16, F32, ROW32, check_rows, norm64, within

pytestmark = pytest.mark.gpu

WIDTHS = [264, 520, 1001, 4100, 8192, 16392, 20000]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def signs(seed, *shape):
    return torch.randint(0, 2, shape, device="cuda", generator=gen(seed)) * 2.0 - 1.0


def check(x, residual, gain, eps, what):
    """Both outputs and the sum; bf16 values below its normal range are off by up to 2^-134."""
    eps = float(torch.tensor(eps, dtype=torch.float32))
    r = vxmoe.add_rms_norm(x, residual, gain, eps, output="both")
    s, v = norm64(x, residual, gain, eps)
    within(r.y, v, v.abs() * (BF16 + 2 * ROW32) + 2.0 ** -134, what + " y")
    check_rows(v, r.q, r.scales, what)
    if residual is not None:
        step, small = (BF16, 2.0 ** -134) if residual.dtype == torch.bfloat16 else (F32, 2.0 ** -150)
        within(r.residual, s, s.abs() * (step + F32) + small, what + " residual")


def residuals(seed, T, d, value):
    """None, and rows of the same magnitude and sign as x, small enough that the sum is finite."""
    return [None] + [(signs(seed, T, d) * value).to(t) for t in (torch.bfloat16, torch.float32)]


@pytest.mark.parametrize("T", [3, 700])
@pytest.mark.parametrize("d", WIDTHS)
def test_squares_above_the_range(T, d):
    gain = (1 + 0.1 * torch.randn(d, device="cuda", generator=gen(2))).bfloat16()
    for big in (3e38, 1e30, 2.0 ** 64):
        x = (signs(1, T, d) * big).bfloat16()
        x[1] = 1.0                     # an ordinary row between
        x[2, d // 2:] = 2.0            # far apart in one row
        for res in residuals(1, T, d, big / 16):
            check(x, res, gain, 1e-6, f"T={T} d={d} {big:.0e}")
            check(x, res, gain, 1e36, f"T={T} d={d} {big:.0e} and a large eps")


@pytest.mark.parametrize("T", [3, 700])
@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -149, 2.0 ** -120, 2.0 ** -101, 2.0 ** -99, 1e-6])
def test_squares_below_the_range(T, d, eps):
    gain = (1 + 0.1 * torch.randn(d, device="cuda", generator=gen(3))).bfloat16()
    wide = gain * 2.0 ** 90
    for power in (-55, -64, -70, -76, -90, -120, -126, -131):
        x = (torch.randn((T, d), device="cuda", generator=gen(4)) * 2.0 ** power).bfloat16()
        for res in residuals(5, T, d, 2.0 ** (power - 1)):
            check(x, res, gain, eps, f"T={T} d={d} 2^{power} eps={eps}")
        check(x, None, wide, eps, f"T={T} d={d} 2^{power} eps={eps} large gains")


@pytest.mark.parametrize("d", WIDTHS)
def test_rows_of_zeros_beside_small_ones(d):
    x = torch.zeros((4, d), device="cuda", dtype=torch.bfloat16)
    x[1, d - 1] = 2.0 ** -133          # the smallest bf16
    x[2] = 2.0 ** -80
    gain = torch.ones(d, device="cuda", dtype=torch.bfloat16)
    r = vxmoe.add_rms_norm(x, None, gain, 0.0, output="both")
    # 0 / 0, as the formula gives it
    assert r.y[[0, 3]].float().isnan().all() and r.scales[[0, 3]].isnan().all()
    check(x[1:3], None, gain, 0.0, "small rows")
    r = vxmoe.add_rms_norm(x, None, gain, 1e-6, output="both")
    assert not r.y[[0, 3]].float().any() and bool((r.scales[[0, 3]] == 2.0 ** -126).all())
