"""grouped_matmul's edge cases in each of its kernels: a few rows, positions as
M (short bank rows, or tens of rows of many experts) and CTA pairs, each with
sorted rows and with gathered ones."""
from __future__ import annotations

import pytest
import torch

import vxmoe
from rows64 import BF16, F32, grouped64, sum_tol, within

pytestmark = pytest.mark.gpu

# positions, experts, outputs, inputs
SHAPES = {"few": (50, 3, 40, 64), "short rows": (300, 3, 96, 128), "tens": (3000, 160, 24, 1040),
          "pairs": (700, 2, 131, 1040)}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(seed, *shape, spread=1.0):
    return (torch.randn(shape, device="cuda", generator=gen(seed)) * spread).bfloat16()


class Case:
    """Operands of one shape; `gather`: positions name rows of half as many."""

    def __init__(self, shape, kind, gather, left=0):
        self.P, self.E, self.N, self.K = SHAPES[shape]
        M = self.P // 2 if gather else self.P
        x, w = normal(1, M, self.K), normal(2, self.E, self.N, self.K, spread=0.05)
        self.kw = {}
        if kind == "e4m3":
            x, w = (x * 20).to(torch.float8_e4m3fn), (w * 400).to(torch.float8_e4m3fn)
            self.kw = dict(x_scales=torch.rand(M, device="cuda", generator=gen(3)) + 0.5,
                           w_scales=torch.rand((self.E, self.N), device="cuda", generator=gen(4)) + 0.5)
        if gather:
            self.kw["rows"] = torch.randint(0, 2 * M, (self.P,), device="cuda", generator=gen(5), dtype=torch.int32)
            self.kw["slots"] = 2
        self.x, self.w = x, w
        # ragged groups, empty ones among them, that end `left` positions early
        cuts = torch.randint(0, self.P - left + 1, (self.E - 1,), device="cuda", generator=gen(6))
        if self.E > 2:
            cuts[1] = cuts[0]
        self.offsets = torch.cat([cuts.new_zeros(1), cuts.sort().values, cuts.new_full((1,), self.P - left)]).int()

    def run(self, x=None, w=None, offsets=None, **kw):
        return vxmoe.grouped_matmul(self.x if x is None else x, self.w if w is None else w,
                                    self.offsets if offsets is None else offsets, **{**self.kw, **kw})

    def check(self, got, what, x=None):
        want, size = grouped64(self.x if x is None else x, self.w, self.offsets, **self.kw)
        within(got[:want.shape[0]], want, want.abs() * (BF16 + 8 * F32) + size * sum_tol(self.K), what)


every = pytest.mark.parametrize("shape", list(SHAPES))
kinds = pytest.mark.parametrize("kind", ["bf16", "e4m3"])
gathers = pytest.mark.parametrize("gather", [False, True])


def bits(t):
    return t.contiguous().view(torch.int16)


@every
@kinds
@gathers
def test_positions_behind_the_last_group(shape, kind, gather):
    c = Case(shape, kind, gather, left=33)
    out = torch.full((c.P + 40, c.N), 7.0, dtype=torch.bfloat16, device="cuda")
    got = c.run(out=out[20:20 + c.P])
    c.check(got, shape)
    assert bool((got[c.P - 33:] == 7).all()) and bool((out[:20] == 7).all()) and bool((out[20 + c.P:] == 7).all())
    if gather:   # what their rows name does not matter
        before = got[:c.P - 33].clone()
        c.kw["rows"][c.P - 33:] = -2 ** 31
        assert torch.equal(bits(c.run(out=out[20:20 + c.P])[:c.P - 33]), bits(before))
        assert bool((got[c.P - 33:] == 7).all())
    out.fill_(3.0)
    c.run(offsets=torch.zeros_like(c.offsets), out=out[20:20 + c.P])
    assert bool((out == 3).all())


@every
@kinds
@gathers
def test_any_offsets(shape, kind, gather):
    """Nothing outside [0, P) is read or written, and offsets count as clamped and ascending."""
    c = Case(shape, kind, gather)
    g = torch.Generator().manual_seed(3)
    for trial in range(6):
        bad = torch.randint(-c.P, 2 * c.P, (c.E + 1,), generator=g).int()
        if trial == 0:
            bad = torch.tensor([0, c.P] * c.E + [0])[:c.E + 1].int()
        if trial == 1:
            bad[:] = -2 ** 31
            bad[-1] = 2 ** 31 - 1
        if trial == 2:
            bad = torch.arange(c.E, -1, -1).int() * (c.P // c.E)
        good = bad.clamp(0, c.P).cummax(0).values
        guard = torch.full((c.P + 64, c.N), 9.0, dtype=torch.bfloat16, device="cuda")
        c.run(offsets=bad.cuda(), out=guard[32:32 + c.P])
        want = torch.full((c.P, c.N), 9.0, dtype=torch.bfloat16, device="cuda")
        c.run(offsets=good.cuda(), out=want)
        assert torch.equal(bits(guard[32:32 + c.P]), bits(want)), f"trial {trial}"
        assert bool((guard[:32] == 9).all()) and bool((guard[32 + c.P:] == 9).all())
        first, last = int(good[0]), int(good[-1])
        assert bool((want[:first] == 9).all()) and bool((want[last:] == 9).all())


@every
@kinds
@gathers
def test_strided_operands(shape, kind, gather):
    c = Case(shape, kind, gather)
    clean = c.run()
    c.check(clean, shape)
    M, K = c.x.shape
    raw = c.x.view(torch.uint8)
    row = raw.shape[1]
    for first in (16, 48, 2, 6):         # rows on 16-byte boundaries, and off them
        wide = torch.full((M, row + 96), 0xFF, dtype=torch.uint8, device="cuda")   # NaN around
        wide[:, first:first + row] = raw
        view = wide.view(c.x.dtype)[:, first // c.x.element_size():][:, :K]
        assert not view.is_contiguous() or M == 1
        assert torch.equal(bits(c.run(x=view)), bits(clean)), f"x from byte {first}"
    assert torch.equal(bits(c.run(x=c.x.t().contiguous().t())), bits(clean)), "columns"
    for left, right in ((16, 16), (4, 8), (1, 6)):
        out = torch.full((c.P, left + c.N + right), 5.0, dtype=torch.bfloat16, device="cuda")
        assert torch.equal(bits(c.run(out=out[:, left:left + c.N])), bits(clean)), f"out from {left}"
        assert bool((out[:, :left] == 5).all()) and bool((out[:, left + c.N:] == 5).all())


@every
@kinds
@gathers
def test_special_values_stay_in_their_group(shape, kind, gather):
    c = Case(shape, kind, gather)
    clean = c.run()
    e = int((c.offsets[1:] - c.offsets[:-1]).argmax())
    mine = torch.zeros(c.P, dtype=torch.bool, device="cuda")
    mine[int(c.offsets[e]):int(c.offsets[e + 1])] = True
    w = c.w.clone()
    w.view(torch.uint8)[e] = 0xFF
    got = c.run(w=w)
    assert got[mine].float().isnan().all() and torch.equal(bits(got[~mine]), bits(clean[~mine]))
    # one row of x: the positions that read it
    row = torch.arange(c.P, device="cuda") if not gather else c.kw["rows"].long() // 2
    bad = int(row[c.P // 3])
    x = c.x.clone()
    x.view(torch.uint8)[bad] = 0xFF
    got = c.run(x=x)
    assert got[row == bad].float().isnan().all() and torch.equal(bits(got[row != bad]), bits(clean[row != bad]))
    # and one that nobody reads
    unread = torch.ones(c.x.shape[0], dtype=torch.bool, device="cuda")
    unread[row] = False
    x = c.x.clone()
    x.view(torch.uint8)[unread] = 0xFF
    assert torch.equal(bits(c.run(x=x)), bits(clean))


@every
@kinds
def test_gathered_rows_on_streams_and_in_graphs(shape, kind):
    """Each call and each graph has its own gathered rows: two of them at once, and one after the other."""
    cases = [Case(shape, kind, True) for _ in range(2)]
    cases[1].kw["rows"] = cases[1].kw["rows"].flip(0).contiguous()
    want = [c.run() for c in cases]
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.run())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    eager = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
                eager[i].append(cases[i].run())
    torch.cuda.synchronize()
    for i in range(2):
        for got in [outs[i]] + eager[i]:
            assert torch.equal(bits(got), bits(want[i]))


@pytest.mark.parametrize("shape", ["few", "short rows", "pairs"])
@gathers
def test_rows_that_lie_gigabytes_apart(shape, gather):
    """Offsets of x and out beyond 32 bits of bytes and of elements."""
    c = Case(shape, "bf16", gather)
    clean = c.run()
    M = c.x.shape[0]
    apart = (5 << 30) // 2 // M // 8 * 8            # elements, 5 GiB in all
    wide = torch.empty(M * apart, dtype=torch.bfloat16, device="cuda").view(M, apart)
    wide[:, :c.K] = c.x
    assert torch.equal(bits(c.run(x=wide[:, :c.K])), bits(clean)), "x"
    del wide
    apart = (5 << 30) // c.P // 8 * 8               # 5 Gi elements
    out = torch.empty(c.P * apart, dtype=torch.bfloat16, device="cuda").view(c.P, apart)
    assert torch.equal(bits(c.run(out=out[:, :c.N])), bits(clean)), "out"
    del out


@pytest.mark.parametrize("P", [9, 2100, 66000])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_a_bank_of_gigabytes(P, kind):
    """The last expert's matrix starts beyond 2^32 elements: few rows, positions as M, CTA pairs."""
    N, K, E = 2048, 2048, 1027
    dtype = torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn
    w = torch.empty((E, N, K), dtype=dtype, device="cuda")
    w[-1:] = normal(1, 1, N, K).to(dtype)
    x = normal(2, P, K).to(dtype)
    kw = {}
    if kind == "e4m3":
        kw = dict(x_scales=torch.rand(P, device="cuda") + 0.5, w_scales=torch.rand((E, N), device="cuda") + 0.5)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offsets[-1] = P
    got = vxmoe.grouped_matmul(x, w, offsets, **kw)
    if kw:
        kw["w_scales"] = kw["w_scales"][-1:]
    want, size = grouped64(x, w[-1:], torch.tensor([0, P]), **kw)
    within(got, want, want.abs() * (BF16 + 8 * F32) + size * sum_tol(K), f"{kind} {P}")
