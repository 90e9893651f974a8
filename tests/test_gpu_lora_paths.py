"""lora_add's edge cases on both of its paths (one launch up to 256 tokens, three
above), with outputs of whole vectors and odd ones."""
from __future__ import annotations

import pytest
import torch

import vxmoe
from rows64 import BF16, lora64, within

pytestmark = pytest.mark.gpu

both = pytest.mark.parametrize("T", [50, 256, 257, 700])
widths = pytest.mark.parametrize("N", [144, 133])


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(seed, *shape, spread=1.0):
    return (torch.randn(shape, device="cuda", generator=gen(seed)) * spread).bfloat16()


def bits(t):
    return t.contiguous().view(torch.int16)


def operands(T, N, K=256, L=3, R=40):
    ids = torch.randint(-1, L, (T,), device="cuda", generator=gen(5), dtype=torch.int32)
    return (normal(1, T, N), normal(2, T, K), normal(3, L, R, K, spread=K ** -0.5), normal(4, L, N, R, spread=R ** -0.5),
            ids)


@both
@widths
def test_special_values_stay_with_their_token_and_adapter(T, N):
    y, x, a, b, ids = operands(T, N)
    ids = torch.arange(T, device="cuda", dtype=torch.int32) % 4 - 1
    clean = vxmoe.lora_add(y, x, a, b, ids)
    x2, a2, y2, b2 = x.clone(), a.clone(), y.clone(), b.clone()
    x2[7] = float("nan")                    # adapter 2
    x2[4] = float("nan")                    # no adapter: x is not read
    a2[1, 3, 5] = float("inf")
    y2[9, 3] = float("inf")
    b2[0, 11, 2] = float("nan")
    got = vxmoe.lora_add(y2, x2, a2, b2, ids)
    keep = (ids != 1)[:, None].expand(T, N).clone()
    keep[7] = False
    keep[9, 3] = False
    keep[ids == 0, 11] = False
    assert torch.equal(got[keep].view(torch.int16), clean[keep].view(torch.int16))
    assert got[7].float().isnan().all() and float(got[9, 3]) == float("inf")
    assert got[ids == 0][:, 11].float().isnan().all() and not got[ids == 1].float().isfinite().any()


@both
@widths
def test_an_infinite_b_gives_no_finite_output(T, N):
    y, x, a, b, ids = operands(T, N)
    clean = vxmoe.lora_add(y, x, a, b, ids)
    b = b.clone()
    b[2, 5, 1] = float("-inf")
    got = vxmoe.lora_add(y, x, a, b, ids)
    hit = torch.zeros((T, N), dtype=torch.bool, device="cuda")
    hit[ids == 2, 5] = True
    assert not got[hit].float().isfinite().any() and torch.equal(got[~hit].view(torch.int16), clean[~hit].view(torch.int16))


@both
@widths
def test_a_token_keeps_its_bits_whatever_the_others_hold(T, N):
    y, x, a, b, ids = operands(T, N)
    whole = vxmoe.lora_add(y, x, a, b, ids)
    kept = torch.arange(T, device="cuda") % 7 == 3
    y2, x2, ids2 = y.flip(0).contiguous(), x.flip(0).contiguous(), ids.roll(5)
    for t, u in ((y2, y), (x2, x), (ids2, ids)):
        t[kept] = u[kept]
    got = vxmoe.lora_add(y2, x2, a, b, ids2)
    assert torch.equal(bits(got[kept]), bits(whole[kept]))


@both
@widths
def test_strided_rows(T, N):
    y, x, a, b, ids = operands(T, N)
    clean = vxmoe.lora_add(y, x, a, b, ids)
    want, tol = lora64(y, x, a, b, ids)
    within(clean, want, want.abs() * BF16 + tol * (1 + BF16), "contiguous")
    for first in (8, 24, 1, 3):
        wide = torch.full((T, x.shape[1] + 40), float("nan"), dtype=torch.bfloat16, device="cuda")
        wide[:, first:first + x.shape[1]] = x
        assert torch.equal(bits(vxmoe.lora_add(y, wide[:, first:first + x.shape[1]], a, b, ids)), bits(clean)), "x"
    for first in (8, 4, 1):
        wide = torch.full((T, N + 40), 5.0, dtype=torch.bfloat16, device="cuda")
        wide[:, first:first + N] = y
        view = wide[:, first:first + N]
        got = vxmoe.lora_add(view, x, a, b, ids)
        assert got.is_contiguous() and torch.equal(bits(got), bits(clean)), "y"
        assert torch.equal(bits(vxmoe.lora_add(view, x, a, b, ids, out=view)), bits(clean)), "in place"
        assert bool((wide[:, :first] == 5).all()) and bool((wide[:, first + N:] == 5).all())
        out = torch.full((T, N + 40), 6.0, dtype=torch.bfloat16, device="cuda")
        assert torch.equal(bits(vxmoe.lora_add(y, x, a, b, ids, out=out[:, first:first + N])), bits(clean)), "out"
        assert bool((out[:, :first] == 6).all()) and bool((out[:, first + N:] == 6).all())


@pytest.mark.parametrize("T", [50, 700])
def test_rows_that_lie_gigabytes_apart(T):
    y, x, a, b, ids = operands(T, 144)
    clean = vxmoe.lora_add(y, x, a, b, ids)
    apart = (5 << 30) // T // 8 * 8                 # 5 Gi elements
    wide = torch.empty(T * apart, dtype=torch.bfloat16, device="cuda").view(T, apart)
    wide[:, :256], wide[:, 1024:1024 + 144] = x, y
    assert torch.equal(bits(vxmoe.lora_add(wide[:, 1024:1024 + 144], wide[:, :256], a, b, ids)), bits(clean))
    vxmoe.lora_add(y, x, a, b, ids, out=wide[:, 2048:2048 + 144])
    assert torch.equal(bits(wide[:, 2048:2048 + 144]), bits(clean))


def test_two_large_batches_at_once_and_a_graph_replayed_on_new_ids():
    calls = [operands(T, 144) for T in (600, 900)]
    streams = [torch.cuda.Stream() for _ in calls]
    want = [vxmoe.lora_add(*c) for c in calls]
    graphs, outs = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(vxmoe.lora_add(*c))
        graphs.append(g)
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    eager = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
                eager[i].append(vxmoe.lora_add(*calls[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for got in [outs[i]] + eager[i]:
            assert torch.equal(bits(got), bits(want[i]))
    for i, (y, x, a, b, ids) in enumerate(calls):    # other requests in the captured call's place
        ids.copy_(ids.flip(0).clone())
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(outs[i]), bits(vxmoe.lora_add(y, x, a, b, ids)))
