"""add_rms_norm and swiglu_e4m3 against their definitions in 64 bits: widths
around every variant (one warp, one CTA, rows read twice, widths no vector
divides), strided and unaligned rows, rows of zeros, NaN and infinities."""
from __future__ import annotations

import pytest
import torch

import vxmoe
from rows64 import BF16, F32, ROW32, check_rows, norm64, swiglu64, within

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(seed, *shape, dtype=torch.bfloat16, spread=1.0):
    return (torch.randn(shape, device="cuda", generator=gen(seed)) * spread).to(dtype)


def check_norm(x, residual, gain, eps, output, what):
    r = vxmoe.add_rms_norm(x, residual, gain, eps, output=output)
    s, v = norm64(x, residual, gain, eps)
    assert (r.y is None) == (output == "e4m3") and (r.q is None) == (output == "bf16") == (r.scales is None)
    if residual is None:
        assert r.residual is None
    else:
        assert r.residual.dtype == residual.dtype and r.residual.shape == x.shape
        step = BF16 if residual.dtype == torch.bfloat16 else F32
        within(r.residual, s, s.abs() * (step + F32), what + " residual")
    if r.y is not None:
        assert r.y.dtype == torch.bfloat16 and r.y.shape == x.shape
        within(r.y, v, v.abs() * (BF16 + 2 * ROW32), what + " y")
    if r.q is not None:
        assert r.q.dtype == torch.float8_e4m3fn and r.q.shape == x.shape and r.scales.shape == x.shape[:-1]
        check_rows(v, r.q, r.scales, what)
    return r


@pytest.mark.parametrize("output", ["bf16", "e4m3", "both"])
@pytest.mark.parametrize("residual", ["none", "bf16", "f32"])
@pytest.mark.parametrize("T,d", [(1, 1), (1, 2048), (5, 8), (7, 127), (3, 128), (4, 129), (6, 256), (5, 264),
                                 (9, 1001), (2, 2560), (2, 4097), (1, 8192), (2, 8200), (1, 16392), (2, 20000)])
def test_norm(T, d, residual, output):
    x = normal(1, T, d, spread=0.7)
    res = None if residual == "none" else normal(2, T, d, spread=3.0,
                                                 dtype=torch.bfloat16 if residual == "bf16" else torch.float32)
    check_norm(x, res, 1 + normal(3, d, spread=0.2), 1e-6, output, f"T={T} d={d} {residual} {output}")


def test_norm_many_rows_and_leading_dimensions():
    x, res = normal(4, 3, 1111, 64), normal(5, 3, 1111, 64)
    check_norm(x, res, normal(6, 64), 1e-5, "both", "3x1111x64")


def test_norm_without_residual_equals_rms_norm():
    """The same formula as rms_norm: one float32 sum in another order, so a
    value may round one bf16 step apart, and most keep their bits."""
    x, gain = normal(7, 33, 2048), 1 + normal(8, 2048, spread=0.1)
    a, b = vxmoe.add_rms_norm(x, None, gain).y, vxmoe.rms_norm(x, gain)
    d = (a.view(torch.int16).int() - b.view(torch.int16).int()).abs()
    assert int(d.max()) <= 1 and float((d == 0).float().mean()) > 0.97


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_strided_and_unaligned_rows(dtype):
    wide = normal(9, 6, 700)
    res = normal(10, 6, 531, dtype=dtype)
    gain = 1 + normal(11, 256, spread=0.2)
    for first in (0, 8, 1, 3):        # 16-byte aligned rows and odd ones
        check_norm(wide[:, first:first + 256], res[:, first:first + 256], gain, 1e-6, "both", f"from {first}")
    check_norm(normal(9, 256, 6).t(), None, gain, 1e-6, "both", "columns")
    check_norm(wide[:1, :256].expand(5, 256), None, gain, 1e-6, "both", "one row repeated")
    check_norm(wide[:, :512][:, ::2], None, gain, 1e-6, "both", "every second element")
    check_norm(wide[:, :256], None, normal(12, 257)[1:], 1e-6, "both", "odd gain")


def test_norm_rows_of_zeros_nan_infinity_and_extremes():
    x = normal(13, 8, 520)
    x[0] = 0
    x[1, 17] = float("nan")
    x[2, 519] = float("inf")
    x[3] = 2.0 ** -130
    x[4] = 3e38                       # the squares leave the float32 range
    x[5, 100:] = 0
    x[6] = torch.finfo(torch.bfloat16).min
    gain = 1 + normal(14, 520, spread=0.1)
    r = vxmoe.add_rms_norm(x, None, gain, 1e-6, output="both")
    y, q = r.y.float(), r.q.float()
    assert not y[0].any() and not q[0].any() and float(r.scales[0]) == 2.0 ** -126
    assert y[1].isnan().all() and q[1].isnan().all() and r.scales[1].isnan()
    assert y[2, 519].isnan() and not y[2, :519].any() and r.scales[2].isnan()
    rows = [3, 4, 5, 6, 7]
    v = norm64(x[rows], None, gain, 1e-6)[1]
    within(r.y[rows], v, v.abs() * (BF16 + 2 * ROW32) + 2.0 ** -134, "y")
    check_rows(v, r.q[rows], r.scales[rows], "extremes")


def test_norm_scales_where_sum_times_gain_leaves_the_range():
    """s * gain overflows (or falls below the normal range) although the
    normalised values do not."""
    x = normal(18, 2, 264) * 2.0 ** 60
    x[1] *= 2.0 ** -120
    gain = normal(19, 264) * 2.0 ** 100
    for row, eps in ((0, 1e-6), (1, 0.0)):
        g = gain if row == 0 else (gain.float() * 2.0 ** -170).bfloat16()
        v = norm64(x[row:row + 1], None, g, eps)[1]
        r = vxmoe.add_rms_norm(x[row:row + 1], None, g, eps, output="e4m3")
        check_rows(v, r.q, r.scales, f"row {row}")


def test_norm_of_nothing():
    r = vxmoe.add_rms_norm(normal(15, 0, 64), normal(16, 0, 64), normal(17, 64), output="both")
    assert r.y.shape == (0, 64) and r.q.shape == (0, 64) and r.scales.shape == (0,) and r.residual.shape == (0, 64)


@pytest.mark.parametrize("P,width", [(1, 1), (3, 17), (640, 512), (5, 128), (4, 131), (9, 640), (2, 661), (2, 4099),
                                     (1, 8192), (2, 9000), (1, 17000)])
def test_swiglu(P, width):
    both = normal(20, P, 2 * width, spread=3.0)
    for gate, up, what in ((both[:, :width], both[:, width:], "halves"),
                           (both[:, :width].contiguous(), both[:, width:].contiguous(), "apart")):
        r = vxmoe.swiglu_e4m3(gate, up)
        assert r.q.shape == (P, width) and r.scales.shape == (P,)
        check_rows(swiglu64(gate, up), r.q, r.scales, f"{P}x{width} {what}")


def test_swiglu_far_gates_and_special_values():
    g = normal(21, 6, 264, spread=2.0)
    u = normal(22, 6, 264)
    g[0] = -87.5                      # e^-87.5 times u stays above 2^-126
    g[1] = -300                       # nothing is left
    g[2] = 300
    g[3, 5] = float("nan")
    u[4, 9] = float("inf")
    g[4, 9] = 1.0
    g[5] = 0
    r = vxmoe.swiglu_e4m3(g, u)
    check_rows(swiglu64(g[:3], u[:3]), r.q[:3], r.scales[:3], "far gates")
    assert r.scales[3].isnan() and r.q[3].float().isnan().all()
    assert r.scales[4].isinf() and r.q[4, 9].float().isnan()
    assert not r.q[5].float().any() and float(r.scales[5]) == 2.0 ** -126


def test_rows_on_another_stream_and_in_a_graph():
    x, res, gain = normal(23, 40, 2048), normal(24, 40, 2048), normal(25, 2048)
    want = vxmoe.add_rms_norm(x, res, gain, output="both")
    wants = vxmoe.swiglu_e4m3(x, res)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = vxmoe.add_rms_norm(x, res, gain, output="both")
        gots = vxmoe.swiglu_e4m3(x, res)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replay = vxmoe.add_rms_norm(x, res, gain, output="both")
        replays = vxmoe.swiglu_e4m3(x, res)
    graph.replay()
    torch.cuda.synchronize()
    for a in (got, replay):
        for u, v in zip(a, want):
            assert torch.equal(u.view(torch.uint8), v.view(torch.uint8))
    for a in (gots, replays):
        for u, v in zip(a, wants):
            assert torch.equal(u.view(torch.uint8), v.view(torch.uint8))


@pytest.mark.parametrize("residual", ["none", "bf16", "f32"])
@pytest.mark.parametrize("T,d", [(3, 2), (3, 4), (5, 130), (5, 252), (700, 12), (3, 258), (3, 516), (2, 1002), (2, 1004),
                                 (2, 8194), (1, 16388)])
def test_norm_widths_that_four_or_two_divide(T, d, residual):
    x = normal(50, T, d, spread=0.7)
    res = None if residual == "none" else normal(51, T, d, spread=3.0,
                                                 dtype=torch.bfloat16 if residual == "bf16" else torch.float32)
    check_norm(x, res, 1 + normal(52, d, spread=0.2), 1e-6, "both", f"T={T} d={d} {residual}")


@pytest.mark.parametrize("first", [1, 2, 4, 6, 8])
def test_rows_that_start_between_vectors(first):
    """One tensor's rows off the others' boundary: the narrowest one counts."""
    T, d = 5, 256
    x, res, gain = normal(53, T, d + 16), normal(54, T, d, dtype=torch.float32), normal(55, d + 16)
    check_norm(x[:, first:first + d], res, 1 + gain[:d], 1e-6, "both", f"x from {first}")
    check_norm(x[:, :d], None, (1 + gain)[first:first + d], 1e-6, "both", f"gain from {first}")
    wide = normal(56, T, d + 16, dtype=torch.float32)
    check_norm(x[:, :d], wide[:, first:first + d], 1 + gain[:d], 1e-6, "both", f"residual from {first}")
    gate, up = normal(57, T, d + 16, spread=2.0), normal(58, T, d)
    r = vxmoe.swiglu_e4m3(gate[:, first:first + d], up)
    check_rows(swiglu64(gate[:, first:first + d], up), r.q, r.scales, f"gate from {first}")


@pytest.mark.parametrize("P,width", [(3, 2), (5, 12), (600, 34), (4, 126), (4, 516), (3, 1002), (2, 8194), (1, 16388)])
def test_swiglu_widths_that_four_or_two_divide(P, width):
    both = normal(59, P, 2 * width, spread=2.0)
    gate, up = both[:, :width], both[:, width:]
    r = vxmoe.swiglu_e4m3(gate, up)
    check_rows(swiglu64(gate, up), r.q, r.scales, f"{P}x{width}")


@pytest.mark.parametrize("width", [201, 402, 612, 401, 802, 777, 1554, 1187, 2374])
def test_many_rows_of_narrow_accesses(width):
    """Enough rows that each takes one warp or few threads, several accesses a thread."""
    T = 2401
    x, res, gain = normal(60, T, width), normal(61, T, width, dtype=torch.float32), 1 + normal(62, width, spread=0.2)
    res[7], x[7] = 0, 0
    x[8, width - 1] = float("nan")
    good = torch.arange(T, device="cuda") != 8
    for residual in (res, res.bfloat16()):
        r = vxmoe.add_rms_norm(x, residual, gain, 1e-6, output="both")
        s, v = norm64(x, residual, gain, 1e-6)
        within(r.y[good], v[good], v[good].abs() * (BF16 + 2 * ROW32), f"{width} y")
        check_rows(v[good], r.q[good], r.scales[good], f"{width} q")
        assert r.y[8].isnan().all() and r.scales[8].isnan()
    both = normal(63, T, 2 * width, spread=2.0)
    q = vxmoe.swiglu_e4m3(both[:, :width], both[:, width:])
    check_rows(swiglu64(both[:, :width], both[:, width:]), q.q, q.scales, f"swiglu {width}")
