"""Refusals of the 8-bit row, grouped and adapter operators that need no GPU:
the C entry points check before they touch the device, and the Python layer
takes CUDA tensors only."""
from __future__ import annotations

import ctypes

import pytest
import torch

P16 = ctypes.c_void_p(1 << 20)      # an aligned address that no refused call reads
ODD = ctypes.c_void_p((1 << 20) + 2)


@pytest.fixture(scope="module")
def lib():
    from vxmoe import _lib
    return _lib.load()


def test_add_rmsnorm_refusals(lib):
    from vxmoe import _lib

    def call(x=P16, ldx=64, res=P16, res_type=0, ldr=64, gain=P16, T=3, d=64, res_out=P16, y=P16, q=P16, scales=P16):
        return lib.vx_add_rmsnorm(x, ldx, res, res_type, ldr, gain, T, d, 1e-6, res_out, y, q, scales, None)

    for kw in (dict(T=-1), dict(d=0), dict(d=(1 << 29) + 8), dict(T=1 << 31), dict(ldx=-1), dict(ldr=-1), dict(x=None), dict(gain=None),
               dict(q=None), dict(scales=None), dict(y=None, q=None, scales=None), dict(res=None),
               dict(res_out=None)):
        assert call(**kw) == _lib.VX_EINVAL_SHAPE, kw
    assert call(res_type=2) == _lib.VX_EINVAL_DTYPE
    assert call(T=0, x=None, gain=None) == _lib.VX_OK


def test_swiglu_e4m3_refusals(lib):
    from vxmoe import _lib

    def call(g=P16, ldg=64, u=P16, ldu=64, rows=3, width=64, q=P16, scales=P16):
        return lib.vx_swiglu_e4m3(g, ldg, u, ldu, rows, width, q, scales, None)

    for kw in (dict(rows=-1), dict(rows=1 << 31), dict(width=0), dict(width=(1 << 29) + 8), dict(ldg=-1), dict(ldu=-1), dict(g=None),
               dict(u=None), dict(q=None), dict(scales=None)):
        assert call(**kw) == _lib.VX_EINVAL_SHAPE, kw
    assert call(rows=0, g=None) == _lib.VX_OK


def test_grouped_matmul_refusals(lib):
    from vxmoe import _lib

    def call(x=P16, dtype=0, x_rows=8, ldx=64, w=P16, xs=None, ws=None, offsets=P16, E=4, N=24, K=64, rows=None,
             slots=1, P=8, out=P16, ldo=24, space=None, nbytes=0):
        return lib.vx_grouped_matmul(x, dtype, x_rows, ldx, w, xs, ws, offsets, E, N, K, rows, slots, P, out, ldo,
                                     space, nbytes, None)

    e4m3 = dict(dtype=2, xs=P16, ws=P16)
    for kw in (dict(E=0), dict(E=2049), dict(N=0), dict(N=(1 << 29) + 1, ldo=1 << 30), dict(K=(1 << 29) + 8, ldx=1 << 30), dict(K=0), dict(K=4, ldx=8), dict(ldx=60), dict(ldx=68),
               dict(slots=0), dict(P=-1), dict(P=1 << 31), dict(x_rows=1 << 31, P=1), dict(x_rows=-1),
               dict(x_rows=7), dict(slots=2), dict(ldo=23), dict(xs=P16), dict(ws=P16), dict(dtype=2),
               dict(dtype=2, xs=P16), dict(K=56, ldx=64, **e4m3), dict(K=48, ldx=56, **e4m3), dict(x=None),
               dict(w=None), dict(offsets=None), dict(out=None), dict(x=ODD), dict(w=ODD),
               dict(rows=P16, x_rows=0)):
        assert call(**kw) == _lib.VX_EINVAL_SHAPE, kw
    assert call(dtype=1) == _lib.VX_EINVAL_DTYPE
    assert call(P=0, x=None, x_rows=0, offsets=None, out=None) == _lib.VX_OK
    assert lib.vx_grouped_matmul_workspace(0, 100000, 4, 64, 0) == 0
    assert lib.vx_grouped_matmul_workspace(0, 8, 4, 64, 1) == 0
    need = lib.vx_grouped_matmul_workspace(0, 100000, 4, 64, 1)
    assert need >= 100000 * 128 and lib.vx_grouped_matmul_workspace(2, 100000, 4, 64, 1) >= 100000 * 68
    for kw in (dict(), dict(space=P16, nbytes=need - 1), dict(space=ODD, nbytes=need)):
        assert call(P=100000, rows=P16, **kw) == _lib.VX_EWORKSPACE, kw
    assert lib.vx_grouped_matmul_workspace(1, 100000, 4, 64, 1) == 0
    assert lib.vx_grouped_matmul_workspace(0, -1, 4, 64, 1) == lib.vx_grouped_matmul_workspace(0, 1, 0, 64, 1) == 0


def test_lora_add_refusals(lib):
    from vxmoe import _lib

    def call(y=P16, ldy=24, x=P16, ldx=64, a=P16, b=P16, ids=P16, L=2, T=3, K=64, N=24, R=8, out=P16, ldo=24, ws=None,
             nbytes=0):
        return lib.vx_lora_add(y, ldy, x, ldx, a, b, ids, None, None, L, T, K, N, R, out, ldo, ws, nbytes, None)

    for kw in (dict(T=-1), dict(T=1 << 31), dict(L=0), dict(L=4097), dict(K=0), dict(K=60), dict(K=(1 << 29) + 8, ldx=1 << 30), dict(N=0),
               dict(N=512 * 65535 + 1, ldy=1 << 26, ldo=1 << 26), dict(R=0), dict(R=12),
               dict(R=264), dict(ldy=23), dict(ldo=23), dict(ldx=63), dict(ldx=68), dict(y=None), dict(x=None),
               dict(a=None), dict(b=None), dict(ids=None), dict(out=None), dict(x=ODD), dict(a=ODD), dict(b=ODD)):
        assert call(**kw) == _lib.VX_EINVAL_SHAPE, kw
    assert call(T=0, x=None, y=None, out=None) == _lib.VX_OK
    need = lib.vx_lora_add_workspace(300, 2, 8)
    assert lib.vx_lora_add_workspace(256, 2, 8) == 0 and need >= 2 * 300 * 4
    for kw in (dict(), dict(ws=P16, nbytes=need - 1), dict(ws=ODD, nbytes=need)):
        assert call(T=300, **kw) == _lib.VX_EWORKSPACE, kw
    assert lib.vx_lora_add_workspace(-1, 2, 8) == lib.vx_lora_add_workspace(300, 0, 8) == 0


def test_python_layer_takes_cuda_tensors_only():
    import vxmoe
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    ids = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: vxmoe.add_rms_norm(x, None, x[0]), lambda: vxmoe.swiglu_e4m3(x, x),
                 lambda: vxmoe.grouped_matmul(x, x[None], ids),
                 lambda: vxmoe.lora_add(x, x, x[None, :1].expand(1, 8, 64), x[None, :, :8], ids)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        vxmoe.add_rms_norm([1.0], None, x[0])
    with pytest.raises(ValueError, match="output"):
        vxmoe.add_rms_norm(x, None, x[0], output="int8")
    with pytest.raises(TypeError):
        vxmoe.grouped_matmul(x.float(), x[None], ids)
