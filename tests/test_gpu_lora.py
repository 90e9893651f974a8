"""lora_add against its definition in 64 bits: batches from one token to many
tiles an adapter, tokens without one, ranks the tenants chose, odd widths,
strided rows, in place."""
from __future__ import annotations

import pytest
import torch

import vxmoe
from rows64 import BF16, lora64, within

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(seed, *shape, spread=1.0):
    return (torch.randn(shape, device="cuda", generator=gen(seed)) * spread).bfloat16()


def operands(T, K, N, L, R, seed=1):
    ids = torch.randint(-1, L, (T,), device="cuda", generator=gen(seed), dtype=torch.int32)
    return (normal(seed + 1, T, N), normal(seed + 2, T, K), normal(seed + 3, L, R, K, spread=K ** -0.5),
            normal(seed + 4, L, N, R, spread=R ** -0.5), ids)


def check(y, x, a, b, ids, what, **kw):
    base = y.clone()
    got = vxmoe.lora_add(y, x, a, b, ids, **kw)
    kw.pop("out", None)
    want, tol = lora64(base, x, a, b, ids.to("cuda"), **kw)
    assert got.dtype == torch.bfloat16 and got.shape == y.shape
    within(got, want, want.abs() * BF16 + tol * (1 + BF16), what)
    none = (ids < 0) | (ids >= a.shape[0])
    assert torch.equal(got[none].view(torch.int16), base[none].view(torch.int16)), "a token without an adapter"
    return got


@pytest.mark.parametrize("T", [1, 2, 16, 17, 65, 300, 1500])
@pytest.mark.parametrize("K,N,L,R", [(64, 64, 3, 8), (2048, 256, 8, 16), (328, 129, 5, 24), (256, 1030, 2, 128),
                                     (128, 72, 70, 64), (512, 520, 1, 256)])
def test_adapters(T, K, N, L, R):
    y, x, a, b, ids = operands(T, K, N, L, R)
    check(y, x, a, b, ids, f"T={T} K={K} N={N} L={L} R={R}")


@pytest.mark.parametrize("T", [1, 40, 700])
def test_ranks_and_scales(T):
    y, x, a, b, ids = operands(T, 640, 320, 9, 48)
    scales = torch.tensor([0.5, -2.0, 0.0, 1.0, 3.0, 0.25, 1e-3, 8.0, 1.5], device="cuda")
    ranks = torch.tensor([48, 1, 7, 8, 9, 47, 33, 0, 16], device="cuda", dtype=torch.int32)
    for r in range(9):      # what lies behind an adapter's rank is not used, whatever it is
        a[r, int(ranks[r]):] = float("nan")
        b[r, :, int(ranks[r]):] = float("inf")
    check(y, x, a, b, ids, f"T={T}", scales=scales, ranks=ranks)
    odd = torch.tensor([99, -5, 7, 8, 9, 47, 33, 0, 16], device="cuda", dtype=torch.int32)
    a, b = normal(5, 9, 48, 640, spread=0.04), normal(6, 9, 320, 48, spread=0.1)
    check(y, x, a, b, ids, f"T={T} clamped", ranks=odd)


@pytest.mark.parametrize("T", [4, 900])
def test_nobody_and_everybody(T):
    y, x, a, b, ids = operands(T, 128, 136, 4, 16)
    for ids in (torch.full((T,), -1), torch.full((T,), 4), torch.full((T,), 2), torch.full((T,), 2**31 - 1),
                torch.full((T,), -2**31), torch.arange(T) % 4, torch.arange(T) * 4 // T):
        ids = ids.to(device="cuda", dtype=torch.int32)
        check(y, x, a, b, ids, "ids")
        check(y, x, a, b, ids.long(), "ids as int64")


def test_special_values_stay_with_their_token_and_adapter():
    y, x, a, b, ids = operands(50, 256, 144, 3, 16)
    ids = torch.arange(50, device="cuda", dtype=torch.int32) % 3
    clean = vxmoe.lora_add(y, x, a, b, ids)
    x2, a2 = x.clone(), a.clone()
    x2[7] = float("nan")
    a2[1, 3, 5] = float("inf")
    y2 = y.clone()
    y2[9, 3] = float("inf")
    got = vxmoe.lora_add(y2, x2, a2, b, ids)
    keep = (ids != 1)
    keep[7] = keep[9] = False
    assert torch.equal(got[keep].view(torch.int16), clean[keep].view(torch.int16))
    assert got[7].float().isnan().all() and float(got[9, 3]) == float("inf")
    assert not got[ids == 1].float().isfinite().any()


def test_strided_rows_and_in_place():
    y, x, a, b, ids = operands(70, 256, 130, 3, 16)
    wide = normal(8, 70, 600)
    check(y, wide[:, 8:264], a, b, ids, "aligned slice")
    check(y, wide[:, 1:257], a, b, ids, "odd slice")
    check(wide[:, 5:135], x, a, b, ids, "odd rows of y")
    check(y.view(7, 10, 130).view(70, 130), x, a, b, ids, "plain")
    got = vxmoe.lora_add(y.view(7, 10, 130), x.view(7, 10, 256), a, b, ids)
    assert got.shape == (7, 10, 130) and torch.equal(got.view(70, 130), vxmoe.lora_add(y, x, a, b, ids))
    out = torch.zeros((70, 300), dtype=torch.bfloat16, device="cuda")
    check(y, x, a, b, ids, "rows of a wider out", out=out[:, 20:150])
    assert not out[:, :20].any() and not out[:, 150:].any()
    want = vxmoe.lora_add(y, x, a, b, ids)
    same = check(y, x, a, b, ids, "in place", out=y)
    assert same.data_ptr() == y.data_ptr() and torch.equal(y, want)


def test_of_nothing():
    y, x, a, b, ids = operands(0, 64, 40, 2, 8)
    assert vxmoe.lora_add(y, x, a, b, ids).shape == (0, 40)


@pytest.mark.parametrize("T", [3, 500])
def test_results_do_not_depend_on_the_batch(T):
    y, x, a, b, ids = operands(T, 512, 264, 5, 32)
    whole = vxmoe.lora_add(y, x, a, b, ids)
    assert torch.equal(whole, vxmoe.lora_add(y, x, a, b, ids))


def test_beside_the_quantised_projection():
    """The shared Q4 projection and the adapters on its output, as a layer calls them."""
    w = vxmoe.MoEWeights.random(num_experts=2, hidden=512, inter=256, shared_inter=256, top_k=1)
    p = w.shared_gate
    _, x, a, b, ids = operands(40, 512, 256, 4, 16)
    y = vxmoe.quantized_matmul(x, p.weight[0], p.scales[0], p.biases[0])
    check(y, x, a, b, ids, "quantized_matmul + lora_add")


def test_two_streams_and_two_graphs_at_once():
    calls = [operands(T, 512, 264, 5, 32, seed=T) for T in (9, 800)]
    want = [vxmoe.lora_add(*c) for c in calls]
    graphs, outs = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(vxmoe.lora_add(*c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in calls]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    eager = []
    for c, s in zip(calls, streams):
        with torch.cuda.stream(s):
            eager.append(vxmoe.lora_add(*c))
    torch.cuda.synchronize()
    for got in (outs, eager):
        for g, v in zip(got, want):
            assert torch.equal(g, v)


@pytest.mark.parametrize("N", [2048, 4096, 4093, 4104])
def test_large_batches_and_wide_outputs(N):
    """Enough items that a CTA takes up to 4,096 outputs, ranks of more than one pass, in place too."""
    y, x, a, b, ids = operands(8200, 64, N, 3, 72, seed=71)
    ranks = torch.tensor([72, 33, 8], device="cuda", dtype=torch.int32)
    got = check(y, x, a, b, ids, f"N={N}", ranks=ranks)
    vxmoe.lora_add(y, x, a, b, ids, ranks=ranks, out=y)
    assert torch.equal(got.view(torch.int16), y.view(torch.int16)), "in place"
