"""swiglu_e4m3 where the gate's exponential alone leaves the float32 range but
the product with up does not."""
from __future__ import annotations

import pytest
import torch

import vxmoe
from rows64 import E4M3, E4M3_SMALL, ROW32, swiglu64, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [8, 264, 777, 1002, 9000])
@pytest.mark.parametrize("g", [-60.0, -88.0, -95.0, -100.0, -104.0, -110.0, -130.0, -150.0, -170.0])
def test_far_negative_gates_with_large_up(g, width):
    T = 5
    gate = torch.full((T, width), g, device="cuda", dtype=torch.bfloat16)
    gate[1, ::2] = 1.5
    gen = torch.Generator("cuda").manual_seed(1)
    # around the size that brings the product back to 1, as far as bf16 goes
    power = min(127.0, -g * 1.4427)
    up = torch.randn((T, width), device="cuda", generator=gen).clamp(-1.9, 1.9).mul(2.0 ** (power - 1)).bfloat16()
    up[2] *= 2.0 ** -20
    up[1, ::2] = 3.0
    # The exponent's argument |g| log2(e) / 2 is rounded twice (the constant and
    # the product, 2^-24 each), a relative |g| / 2 * 2^-23 of its exponential,
    # which enters twice: |g| 2^-23; the rest as in ROW32.
    rel = ROW32 - 2.0 ** -23 * g
    v = swiglu64(gate, up)
    want = v.abs().amax(-1).div(448).clamp_min(2.0 ** -126)
    r = vxmoe.swiglu_e4m3(gate, up)
    within(r.scales, want, rel * want, f"{g} scales")
    t = v / want[:, None]
    within(r.q.float(), t, t.abs() * (E4M3 + 2 * rel) + E4M3_SMALL, f"{g} q")
