"""Products over more inputs than their kernels' bounded waits allow for are
refused before anything is launched."""
from __future__ import annotations

import ctypes

import pytest

P16 = ctypes.c_void_p(1 << 20)      # an aligned address that no refused call reads


@pytest.mark.parametrize("K", [(1 << 24) + 16, 1 << 25, 1 << 29])
def test_inputs_beyond_the_waits(K):
    from vxmoe import _lib
    lib = _lib.load()
    for dtype, scales in ((_lib.VX_DTYPE_BF16, None), (_lib.VX_DTYPE_E4M3, P16)):
        assert lib.vx_grouped_matmul(P16, dtype, 100, K, P16, scales, scales, P16, 1, 16, K, None, 1, 100, P16, 16, None,
                                     0, None) == _lib.VX_EINVAL_SHAPE
    assert lib.vx_lora_add(P16, 16, P16, K, P16, P16, P16, None, None, 1, 3, K, 16, 8, P16, 16, None, 0,
                           None) == _lib.VX_EINVAL_SHAPE
