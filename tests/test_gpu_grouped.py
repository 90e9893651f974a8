"""grouped_matmul against its definition in 64 bits: ragged groups from empty
to several tiles, odd outputs, every kind of row order, strided operands,
positions behind the last group, bad offsets and rows."""
from __future__ import annotations

import pytest
import torch

import vxmoe
from rows64 import BF16, F32, grouped64, sum_tol, within

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(seed, *shape, spread=1.0):
    return (torch.randn(shape, device="cuda", generator=gen(seed)) * spread).bfloat16()


def operands(kind, M, E, N, K, seed=1):
    """x, w and their scales (None for bf16)."""
    x, w = normal(seed, M, K), normal(seed + 1, E, N, K, spread=0.05)
    if kind == "bf16":
        return x, w, None, None
    xs = torch.rand(M, device="cuda", generator=gen(seed + 2)) + 0.5
    ws = torch.rand((E, N), device="cuda", generator=gen(seed + 3)) * 0.02 + 0.01
    return (x * 20).to(torch.float8_e4m3fn), (w * 400).to(torch.float8_e4m3fn), xs, ws


def offsets_of(counts):
    c = torch.tensor([0] + list(counts), device="cuda").cumsum(0)
    return c.int()


def check(x, w, offsets, what, **kw):
    got = vxmoe.grouped_matmul(x, w, offsets, **kw)
    kw.pop("out", None)
    want, size = grouped64(x, w, offsets, **kw)
    assert got.dtype == torch.bfloat16
    within(got[:want.shape[0]], want, want.abs() * (BF16 + 8 * F32) + size * sum_tol(x.shape[1]), what)
    return got


COUNTS = [
    [1], [0, 0, 3, 0], [16, 17, 31, 32, 33], [0, 255, 256, 257, 0, 1], [300, 5, 700], [1] * 40, [513, 0, 0, 2],
]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c[:8])))
@pytest.mark.parametrize("N,K", [(96, 64), (257, 208), (300, 1024)])
def test_sorted_rows(kind, counts, N, K):
    P = sum(counts)
    x, w, xs, ws = operands(kind, P, len(counts), N, K)
    check(x, w, offsets_of(counts), f"{kind} {counts} {N}x{K}", x_scales=xs, w_scales=ws)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("N", [1, 2, 7, 8, 127, 128, 129, 255, 256, 511, 640])
@pytest.mark.parametrize("K", [16, 48, 64, 80, 128])
def test_odd_outputs_and_inputs(kind, N, K):
    x, w, xs, ws = operands(kind, 45, 3, N, K)
    check(x, w, offsets_of([20, 4, 21]), f"{kind} {N}x{K}", x_scales=xs, w_scales=ws)


def routed(T, E, k, seed):
    ids = torch.rand((T, E), device="cuda", generator=gen(seed)).topk(k, dim=1).indices.int()
    return ids, vxmoe.permute(ids, E)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("T,E,k,N,K", [(1, 32, 10, 128, 256), (1, 1, 1, 65, 64), (64, 128, 10, 264, 512),
                                       (300, 16, 4, 130, 144), (2000, 8, 2, 256, 64), (37, 512, 10, 32, 128)])
def test_routed_rows(kind, T, E, k, N, K):
    x, w, xs, ws = operands(kind, T, E, N, K, seed=5)
    _, p = routed(T, E, k, 6)
    check(x, w, p.offsets, f"{kind} T={T} E={E}", rows=p.order, slots=k, x_scales=xs, w_scales=ws)


def test_rows_without_slots_and_the_same_row_often():
    x, w, _, _ = operands("bf16", 9, 4, 72, 96)
    rows = torch.tensor([8, 8, 8, 0, 1, 0, 5, 5, 2, 3], device="cuda", dtype=torch.int32)
    check(x, w, offsets_of([3, 0, 5, 2]), "rows", rows=rows)
    check(x, w, offsets_of([3, 0, 5, 2]), "rows as int64", rows=rows.long())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("gather", [False, True])
def test_positions_behind_the_last_group_are_left(kind, gather):
    x, w, xs, ws = operands(kind, 50, 3, 40, 64)
    rows = torch.randint(0, 50, (50,), device="cuda", generator=gen(7), dtype=torch.int32) if gather else None
    out = torch.full((50, 40), 7.0, dtype=torch.bfloat16, device="cuda")
    offsets = offsets_of([5, 0, 12])
    got = check(x, w, offsets, f"{kind} {gather}", rows=rows, x_scales=xs, w_scales=ws, out=out)
    assert got.data_ptr() == out.data_ptr() and bool((out[17:] == 7).all())
    out.fill_(3.0)
    vxmoe.grouped_matmul(x, w, torch.zeros(4, dtype=torch.int32, device="cuda"), rows=rows, x_scales=xs,
                         w_scales=ws, out=out)
    assert bool((out == 3).all())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("P,E,K", [(9, 4, 64), (300, 2, 528), (40, 1, 64)])
def test_bad_offsets_touch_only_what_they_may(kind, P, E, K):
    """Any offsets: nothing outside [0, P) is read or written, no position twice."""
    x, w, xs, ws = operands(kind, P, E, 48, K)
    g = torch.Generator().manual_seed(3)
    for trial in range(12):
        bad = torch.randint(-P, 2 * P, (E + 1,), generator=g).int()
        if trial == 0:
            bad = torch.tensor([0, P] * E + [0])[:E + 1].int()
        if trial == 1:
            bad[:] = -2**31
            bad[-1] = 2**31 - 1
        good = bad.clamp(0, P).cummax(0).values
        guard = torch.full((P + 64, 48), 9.0, dtype=torch.bfloat16, device="cuda")
        out = guard[32:32 + P]
        vxmoe.grouped_matmul(x, w, bad.cuda(), x_scales=xs, w_scales=ws, out=out)
        want = torch.full((P, 48), 9.0, dtype=torch.bfloat16, device="cuda")
        vxmoe.grouped_matmul(x, w, good.cuda(), x_scales=xs, w_scales=ws, out=want)
        assert torch.equal(out, want), f"{bad.tolist()}"
        assert bool((guard[:32] == 9).all()) and bool((guard[32 + P:] == 9).all())
        first, last = int(good[0]), int(good[-1])
        assert bool((want[:first] == 9).all()) and bool((want[last:] == 9).all())


def test_offsets_and_rows_out_of_range():
    """Offsets are clamped to [0, P] and to ascend; a row outside x gives zeros."""
    x, w, _, _ = operands("bf16", 20, 4, 24, 64)
    out = torch.full((20, 24), 5.0, dtype=torch.bfloat16, device="cuda")
    bad = torch.tensor([-3, 6, 4, 1000, 30], dtype=torch.int32, device="cuda")
    vxmoe.grouped_matmul(x, w, bad, out=out)
    want, size = grouped64(x, w, torch.tensor([0, 6, 6, 20, 20]))
    # expert 1 has the descending pair [6, 4): nothing; expert 2 goes on from 6
    again, size2 = grouped64(x[4:], w[2:3], torch.tensor([0, 16]))
    got = out.double()
    tol = sum_tol(64)
    for lo, hi, ref, sz in ((0, 4, want[:4], size[:4]), (6, 20, again[2:], size2[2:])):
        within(got[lo:hi], ref, ref.abs() * (BF16 + 8 * F32) + sz * tol, f"{lo}:{hi}")
    rows = torch.tensor([0, 99, -1, 3, 20, 2**31 - 1, -2**31], dtype=torch.int32, device="cuda")
    for kind in ("bf16", "e4m3"):
        x, w, xs, ws = operands(kind, 20, 1, 24, 64)
        x.view(torch.uint8)[1] = 0xFF          # a row of NaN that no position names
        got = vxmoe.grouped_matmul(x, w, offsets_of([7]), rows=rows, x_scales=xs, w_scales=ws)
        assert not got[[1, 2, 4, 5, 6]].float().any()
        assert got[[0, 3]].float().isfinite().all()


def test_a_group_does_not_see_its_neighbours():
    """NaN and infinities in one expert's rows or bank stay there."""
    for kind in ("bf16", "e4m3"):
        x, w, xs, ws = operands(kind, 60, 3, 80, 128)
        clean = vxmoe.grouped_matmul(x, w, offsets_of([20, 7, 33]), x_scales=xs, w_scales=ws)
        x2, w2 = x.clone(), w.clone()
        x2.view(torch.uint8)[20:27] = 0xFF
        w2.view(torch.uint8)[1] = 0xFF
        got = vxmoe.grouped_matmul(x2, w2, offsets_of([20, 7, 33]), x_scales=xs, w_scales=ws)
        keep = torch.ones(60, dtype=torch.bool, device="cuda")
        keep[20:27] = False
        assert got[20:27].float().isnan().all()
        assert torch.equal(got[keep].view(torch.int16), clean[keep].view(torch.int16))


def test_strided_operands():
    x, w, _, _ = operands("bf16", 33, 2, 50, 128)
    wide = normal(9, 33, 300)
    offsets = offsets_of([20, 13])
    out = torch.zeros((33, 90), dtype=torch.bfloat16, device="cuda")
    for view, what in ((wide[:, 8:136], "aligned slice"), (wide[:, 3:131], "odd slice"),
                       (wide[:1, :128].expand(33, 128), "one row repeated"),
                       (normal(10, 128, 33).t(), "columns")):
        check(view, w, offsets, what)
    check(x, w, offsets, "rows of a wider out", out=out[:, 20:70])
    assert not out[:, :20].any() and not out[:, 70:].any()
    check(x, w, offsets, "odd out", out=out[:, 1:51])


def test_nothing_to_do():
    x, w, _, _ = operands("bf16", 0, 2, 50, 64)
    assert vxmoe.grouped_matmul(x, w, offsets_of([0, 0])).shape == (0, 50)
    x, w, _, _ = operands("bf16", 4, 2, 50, 64)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert vxmoe.grouped_matmul(x, w, offsets_of([0, 0]), rows=none).shape == (0, 50)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("counts", [[390, 10], [3, 1], [60, 0]])
def test_calls_repeat_and_rows_do_not_depend_on_their_neighbours(kind, counts):
    """The same call gives the same bits, whatever the other rows of its groups hold."""
    x, w, xs, ws = operands(kind, sum(counts), 2, 144, 320)
    whole = vxmoe.grouped_matmul(x, w, offsets_of(counts), x_scales=xs, w_scales=ws)
    again = vxmoe.grouped_matmul(x, w, offsets_of(counts), x_scales=xs, w_scales=ws)
    assert torch.equal(whole, again)
    other = x.flip(0).contiguous()
    keep = counts[0] // 2
    other[keep] = x[keep]
    if xs is not None:
        xs = xs.flip(0).contiguous()
        xs[keep] = operands(kind, sum(counts), 2, 144, 320)[2][keep]
    mixed = vxmoe.grouped_matmul(other, w, offsets_of(counts), x_scales=xs, w_scales=ws)
    assert torch.equal(mixed[keep], whole[keep])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("counts", [[140], [129, 300], [256, 257, 512, 1, 0, 700], [1100, 3]],
                         ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("N", [1, 127, 130, 257, 512, 636])
def test_many_rows(kind, counts, N):
    """More than 128 rows an expert and rows of more than 512 bytes: the CTA pairs' tiles,
    sorted rows and gathered ones, odd and wider out, special values in another group."""
    K, P = 528 if kind == "e4m3" else 264, sum(counts)
    x, w, xs, ws = operands(kind, P, len(counts), N, K, seed=21)
    offsets = offsets_of(counts)
    clean = check(x, w, offsets, f"{kind} {counts} N={N}", x_scales=xs, w_scales=ws)
    rows = torch.randint(0, 2 * P, (P,), device="cuda", generator=gen(22), dtype=torch.int32)
    check(x, w, offsets, f"{kind} {counts} N={N} rows", rows=rows, slots=2, x_scales=xs, w_scales=ws)
    out = torch.full((P, N + 9), 5.0, dtype=torch.bfloat16, device="cuda")
    check(x, w, offsets, f"{kind} {counts} N={N} out", x_scales=xs, w_scales=ws, out=out[:, 3:3 + N])
    assert bool((out[:, :3] == 5).all()) and bool((out[:, 3 + N:] == 5).all())
    if len(counts) > 1:
        x2, w2 = x.clone(), w.clone()
        x2.view(torch.uint8)[:counts[0]] = 0xFF
        w2.view(torch.uint8)[0] = 0xFF
        got = vxmoe.grouped_matmul(x2, w2, offsets, x_scales=xs, w_scales=ws)
        assert got[:counts[0]].float().isnan().all()
        assert torch.equal(got[counts[0]:].view(torch.int16), clean[counts[0]:].view(torch.int16))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("counts", [[70], [64, 65], [0, 63, 128, 129, 17, 0, 1], [i * 37 % 97 for i in range(160)],
                                    [(0, 64, 65, 1, 128, 129, 16, 15)[i % 8] for i in range(152)]],
                         ids=lambda c: f"{len(c)}-" + "-".join(map(str, c[:8])))
@pytest.mark.parametrize("N", [1, 127, 130, 256, 272, 636])
def test_tens_of_rows(kind, counts, N):
    """Tiles of up to 64 and up to 128 positions, with enough experts for them and without."""
    K, P = 272, sum(counts)
    x, w, xs, ws = operands(kind, P, len(counts), N, K, seed=23)
    offsets = offsets_of(counts)
    clean = check(x, w, offsets, f"{kind} {counts} N={N}", x_scales=xs, w_scales=ws)
    rows = torch.randint(0, 3 * P, (P,), device="cuda", generator=gen(24), dtype=torch.int32)
    check(x, w, offsets, f"{kind} {counts} N={N} rows", rows=rows, slots=3, x_scales=xs, w_scales=ws)
    for wide in (9, 16):
        out = torch.full((P, N + wide + 16 - N % 16), 5.0, dtype=torch.bfloat16, device="cuda")
        got = check(x, w, offsets, f"{kind} {counts} N={N} out", x_scales=xs, w_scales=ws, out=out[:, wide:wide + N])
        assert bool((out[:, :wide] == 5).all()) and bool((out[:, wide + N:] == 5).all())
        assert torch.equal(got.contiguous().view(torch.int16), clean.view(torch.int16))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("E,P", [(1, 1), (1, 8), (3, 12), (40, 37), (512, 10), (512, 700), (2048, 9)])
@pytest.mark.parametrize("N,K", [(16, 64), (33, 176), (1000, 2048), (128, 4112)])
def test_few_rows(kind, E, P, N, K):
    """Groups around the few-rows kernel's items of 8, one warp and eight to a unit."""
    if E * N * K > 1 << 28:
        N = max(1, (1 << 28) // (E * K))
    x, w, xs, ws = operands(kind, 5, E, N, K, seed=11)
    ids = torch.randint(0, E, (P,), device="cuda", generator=gen(12))
    if P > 30:
        ids[:11] = E // 2          # a group of more than one item
    ids = ids.sort().values
    offsets = torch.cat([ids.new_zeros(1), torch.bincount(ids, minlength=E).cumsum(0)]).int()
    rows = torch.randint(0, 10, (P,), device="cuda", generator=gen(13), dtype=torch.int32)
    check(x, w, offsets, f"{kind} E={E} P={P} {N}x{K}", rows=rows, slots=2, x_scales=xs, w_scales=ws)


def test_two_streams_and_two_graphs_at_once():
    x, w, _, _ = operands("bf16", 700, 16, 264, 512)
    counts = offsets_of([44] * 12 + [0, 1, 170, 1])
    want = vxmoe.grouped_matmul(x, w, counts)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(vxmoe.grouped_matmul(x, w, counts))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    eager = []
    for s in streams:
        with torch.cuda.stream(s):
            eager.append(vxmoe.grouped_matmul(x, w, counts))
    torch.cuda.synchronize()
    for got in outs + eager:
        assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("K", [256, 576])
@pytest.mark.parametrize("counts", [[100], [5, 128, 127, 66], [17] * 12, [300, 0, 1000, 33]],
                         ids=lambda c: "-".join(map(str, c[:4])))
@pytest.mark.parametrize("N", [4, 12, 20, 131, 258, 260, 268, 304])
def test_stores_of_every_width(kind, K, counts, N):
    """Short bank rows (the positions-as-M tiles) and longer ones; outputs whose rows
    16, 4, 2 or 1 elements divide, with and without neighbours in the same row."""
    P = sum(counts)
    x, w, xs, ws = operands(kind, P, len(counts), N, K, seed=31)
    offsets = offsets_of(counts)
    what = f"{kind} {counts} {N}x{K}"
    clean = check(x, w, offsets, what, x_scales=xs, w_scales=ws)
    for left, width in ((0, 320), (4, 324), (3, 331)):
        out = torch.full((P + 2, width), 5.0, dtype=torch.bfloat16, device="cuda")
        got = vxmoe.grouped_matmul(x, w, offsets, x_scales=xs, w_scales=ws, out=out[1:P + 1, left:left + N])
        assert torch.equal(got.contiguous().view(torch.int16), clean.view(torch.int16)), f"{what} from {left}"
        out[1:P + 1, left:left + N] = 5
        assert bool((out == 5).all()), f"{what}: something beside the outputs was written"
