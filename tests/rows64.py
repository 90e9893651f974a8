"""Plain 64-bit forms of the 8-bit row, grouped and adapter operators, and the
bounds their outputs are held to.

A rounding is off by at most half a step: relative 2^-8 for bf16, 2^-4 for
e4m3 (2^-10 absolute below its smallest normal value), 2^-24 for float32.
"""
from __future__ import annotations

import torch

BF16, E4M3, F32 = 2.0 ** -8, 2.0 ** -4, 2.0 ** -24
E4M3_SMALL = 2.0 ** -10
# float32 arithmetic of one row: at most 40 additions in a thread, 5 in its
# warp and 32 over the warps (half of it after the square root), then about
# eight more roundings: under 64 * 2^-24
ROW32 = 64 * F32


def bf16(t):
    return t.to(torch.bfloat16)


def within(got, want, tol, what):
    """|got - want| <= tol elementwise in float64; NaN and infinities equal."""
    got, want = got.double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN places differ"
    odd = ~fine & ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd]), f"{what}: infinities differ"
    off = ((got - want).abs() - tol)[fine]
    assert not off.numel() or float(off.max()) <= 0, f"{what}: over the bound by {float(off.max()):.3g}"


def norm64(x, residual, gain, eps):
    s = x.double() + (0 if residual is None else residual.double())
    return s, s / (s.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double()


def swiglu64(gate, up):
    g = gate.double()
    return g / (1 + torch.exp(-g)) * up.double()


def check_rows(v, q, scales, what):
    """e4m3 rows of the 64-bit values v: scale max|v| / 448 (at least 2^-126),
    q the nearest value of v / scale."""
    want = v.abs().amax(-1).div(448).clamp_min(2.0 ** -126)
    within(scales, want, ROW32 * want, f"{what} scales")
    t = v / want[..., None]
    within(q.float(), t, t.abs() * (E4M3 + 2 * ROW32) + E4M3_SMALL, f"{what} q")


def grouped64(x, w, offsets, rows=None, slots=1, x_scales=None, w_scales=None):
    """(out, sum of the terms' magnitudes) for the positions below offsets[-1]."""
    bounds = offsets.tolist()
    P = bounds[-1]
    r = torch.arange(P, device=x.device) if rows is None else rows.long()[:P] // slots
    xd = x.double() * (1 if x_scales is None else x_scales.double()[:, None])
    out = torch.zeros((P, w.shape[1]), dtype=torch.float64, device=x.device)
    size = torch.zeros_like(out)
    for e, (i, j) in enumerate(zip(bounds, bounds[1:])):
        we = w[e].double() * (1 if w_scales is None else w_scales[e].double()[:, None])
        out[i:j] = xd[r[i:j]] @ we.T
        size[i:j] = xd[r[i:j]].abs() @ we.abs().T
    return out, size


def sum_tol(K):
    """A float32 sum of K products on the tensor cores, relative to the sum of
    their magnitudes: one truncation (2^-23) for each block of 16 inputs that
    joins the accumulator, and the alignment of the 16 terms inside a block."""
    return (K / 16 + 16) * 2.0 ** -23


def lora64(y, x, a, b, adapters, scales=None, ranks=None):
    """(out, bound of the error of its sums before the last rounding)."""
    out = y.double().clone()
    tol = torch.zeros_like(out)
    L, R, K = a.shape
    for e in range(L):
        at = (adapters == e).nonzero()[:, 0]
        r = R if ranks is None else max(0, min(R, int(ranks[e])))
        if not at.numel() or not r:
            continue
        s = 1.0 if scales is None else float(scales[e])
        xd, ad, bd = x[at].double(), a[e, :r].double(), b[e, :, :r].double()
        h = xd @ ad.T
        out[at] += s * (h @ bd.T)
        # the inner values: a float32 sum of K products, then 16 bits or more
        # on the way to the second product (2^-16); the second sum
        dh = sum_tol(K) * (xd.abs() @ ad.abs().T) + 2.0 ** -16 * h.abs()
        tol[at] += abs(s) * ((dh + sum_tol(r) * h.abs()) @ bd.abs().T)
    return out, tol + F32 * 4 * out.abs()
