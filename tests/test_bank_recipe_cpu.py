"""The integration guide's quantisation of a bank to 8 bits, as it stands there:
types that grouped_matmul takes, rows of zeros and of the smallest values."""
from __future__ import annotations

import os
import re

import pytest
import torch

from rows64 import E4M3, E4M3_SMALL, F32

GUIDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_recipe(dtype):
    with open(GUIDE) as f:
        text = f.read()
    block = re.search(r"is quantised once at load(?:(?!```|\n#).)*```python\n(.*?)```", text, re.S).group(1)
    w = (torch.randn((3, 5, 32), generator=torch.Generator().manual_seed(1)) * 0.05).to(dtype)
    w[1, 2] = 0
    w[2, 4] = torch.finfo(dtype).smallest_normal
    w[0, 0, 1:] = 0
    names = {"torch": torch, "w": w}
    exec(block, names)
    q, scales = names["q"], names["scales"]
    assert q.dtype == torch.float8_e4m3fn and q.shape == w.shape
    assert scales.dtype == torch.float32 and scales.shape == w.shape[:-1]
    v, s = q.double(), scales.double()
    assert v.isfinite().all() and bool((s >= 2.0 ** -126).all()) and not v[1, 2].any()
    # one rounding to e4m3 of w / scale, the scale's and the quotient's in float32
    t = w.double() / s[..., None]
    assert bool(((v - t).abs() <= t.abs() * (E4M3 + 2 * F32) + E4M3_SMALL).all())
    assert bool((t.abs().amax(-1) <= 448 * (1 + 2 * F32)).all())
