"""The operators around the experts in the order a layer calls them: the norm
with the residual's addition, the router, the expert sort, the grouped
gate/up product over 8-bit (or bf16) banks, SwiGLU, the grouped down product,
the score-weighted combine; each stage against 64 bits on what it was given,
and the whole chain captured into a CUDA graph."""
from __future__ import annotations

import pytest
import torch

import vxmoe
from rows64 import BF16, F32, ROW32, check_rows, grouped64, norm64, sum_tol, swiglu64, within

pytestmark = pytest.mark.gpu


def bank(E, N, K, seed):
    """A bf16 bank, and its 8-bit rows with one scale per output."""
    w = torch.randn((E, N, K), device="cuda", generator=torch.Generator("cuda").manual_seed(seed)) * 0.05
    scale = w.abs().amax(-1) / 448
    return w.bfloat16(), (w / scale[..., None]).to(torch.float8_e4m3fn), scale


def layer(x, res, gain, router_w, gu, down, kind, k):
    """One expert layer; every stage's output."""
    E, d = router_w.shape
    I = gu[0].shape[1] // 2
    r = vxmoe.add_rms_norm(x, res, gain, output="both" if kind == "e4m3" else "bf16")
    route = vxmoe.route(r.y, router_w, k)
    p = vxmoe.permute(route.inds, E)
    if kind == "e4m3":
        h = vxmoe.grouped_matmul(r.q, gu[1], p.offsets, rows=p.order, slots=k, x_scales=r.scales, w_scales=gu[2])
        a = vxmoe.swiglu_e4m3(h[:, :I], h[:, I:])
        o = vxmoe.grouped_matmul(a.q, down[1], p.offsets, x_scales=a.scales, w_scales=down[2])
    else:
        h = vxmoe.grouped_matmul(r.y, gu[0], p.offsets, rows=p.order, slots=k)
        a = vxmoe.swiglu(h[:, :I], h[:, I:])
        o = vxmoe.grouped_matmul(a, down[0], p.offsets)
    slots = o[p.inverse.long()].view(-1, k, d)
    y = (slots.float() * route.weights.float()[..., None]).sum(1) + r.residual.float()
    return r, route, p, h, a, o, y


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("T", [1, 3, 64, 700])
def test_expert_layer(kind, T):
    E, d, I, k = 32, 512, 160, 4
    g = torch.Generator("cuda").manual_seed(T)
    x = torch.randn((T, d), device="cuda", generator=g).bfloat16()
    res = torch.randn((T, d), device="cuda", generator=g) * 3
    gain = (1 + 0.1 * torch.randn(d, device="cuda", generator=g)).bfloat16()
    router_w = (torch.randn((E, d), device="cuda", generator=g) * 0.05).bfloat16()
    gu, down = bank(E, 2 * I, d, 1), bank(E, d, I, 2)
    r, route, p, h, a, o, y = layer(x, res, gain, router_w, gu, down, kind, k)
    s, v = norm64(x, res, gain, 1e-6)
    within(r.residual, s, s.abs() * 2 * F32, "residual")
    within(r.y, v, v.abs() * (BF16 + 2 * ROW32), "norm")
    if kind == "e4m3":
        check_rows(v, r.q, r.scales, "norm")
        want, size = grouped64(r.q, gu[1], p.offsets, p.order, k, r.scales, gu[2])
    else:
        want, size = grouped64(r.y, gu[0], p.offsets, p.order, k)
    within(h, want, want.abs() * (BF16 + 8 * F32) + size * sum_tol(d), "gate/up")
    if kind == "e4m3":
        check_rows(swiglu64(h[:, :I], h[:, I:]), a.q, a.scales, "swiglu")
        want, size = grouped64(a.q, down[1], p.offsets, x_scales=a.scales, w_scales=down[2])
    else:
        want, size = grouped64(a, down[0], p.offsets)
    within(o, want, want.abs() * (BF16 + 8 * F32) + size * sum_tol(I), "down")

    again = layer(x, res, gain, router_w, gu, down, kind, k)[-1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer(x, res, gain, router_w, gu, down, kind, k)[-1]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, y) and torch.equal(captured, y)
