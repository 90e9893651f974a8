"""What the Python layer of the 8-bit row, grouped and adapter operators
refuses, and on which exception."""
from __future__ import annotations

import pytest
import torch

import vxmoe

pytestmark = pytest.mark.gpu


def bf(*shape):
    return torch.ones(shape, dtype=torch.bfloat16, device="cuda")


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def f8(*shape):
    return bf(*shape).to(torch.float8_e4m3fn)


def f32(*shape):
    return torch.ones(shape, device="cuda")


@pytest.mark.parametrize("error,call", [
    (TypeError, lambda: vxmoe.add_rms_norm(f32(2, 8), None, bf(8))),
    (TypeError, lambda: vxmoe.add_rms_norm(bf(2, 8), None, f32(8))),
    (TypeError, lambda: vxmoe.add_rms_norm(bf(2, 8), bf(2, 8).half(), bf(8))),
    (ValueError, lambda: vxmoe.add_rms_norm(bf(2, 8), bf(3, 8), bf(8))),
    (ValueError, lambda: vxmoe.add_rms_norm(bf(2, 8), bf(8), bf(8))),
    (ValueError, lambda: vxmoe.add_rms_norm(bf(2, 8), None, bf(9))),
    (ValueError, lambda: vxmoe.add_rms_norm(bf(2, 0), None, bf(0))),
    (ValueError, lambda: vxmoe.add_rms_norm(bf(2, 8), bf(2, 8).cpu(), bf(8))),
    (TypeError, lambda: vxmoe.swiglu_e4m3(bf(2, 8), f32(2, 8))),
    (ValueError, lambda: vxmoe.swiglu_e4m3(bf(2, 8), bf(2, 9))),
    (ValueError, lambda: vxmoe.swiglu_e4m3(bf(2, 0), bf(2, 0))),
    (TypeError, lambda: vxmoe.grouped_matmul(f32(2, 16), f32(1, 4, 16), i32(0, 2))),
    (TypeError, lambda: vxmoe.grouped_matmul(bf(2, 16), f8(1, 4, 16), i32(0, 2))),
    (TypeError, lambda: vxmoe.grouped_matmul(bf(2, 16), bf(1, 4, 16), f32(2))),
    (ValueError, lambda: vxmoe.grouped_matmul(bf(2, 16), bf(1, 4, 24), i32(0, 2))),
    (ValueError, lambda: vxmoe.grouped_matmul(bf(2, 2, 16), bf(1, 4, 16), i32(0, 2))),
    (ValueError, lambda: vxmoe.grouped_matmul(bf(2, 16), bf(4, 16), i32(0, 2))),
    (ValueError, lambda: vxmoe.grouped_matmul(bf(2, 16), bf(1, 16, 4).transpose(1, 2), i32(0, 2))),
    (ValueError, lambda: vxmoe.grouped_matmul(bf(2, 12), bf(1, 4, 12), i32(0, 2))),
    (ValueError, lambda: vxmoe.grouped_matmul(bf(2, 16), bf(65)[1:].view(1, 4, 16), i32(0, 2))),
    (ValueError, lambda: vxmoe.grouped_matmul(bf(2, 16), bf(1, 4, 16), i32(0, 1, 2))),
    (ValueError, lambda: vxmoe.grouped_matmul(bf(2, 16), bf(1, 4, 16), i32(0, 2), slots=2)),
    (ValueError, lambda: vxmoe.grouped_matmul(bf(2, 16), bf(1, 4, 16), i32(0, 2), rows=i32(0, 1), slots=0)),
    (ValueError, lambda: vxmoe.grouped_matmul(bf(0, 16), bf(1, 4, 16), i32(0, 2), rows=i32(0, 1))),
    (ValueError, lambda: vxmoe.grouped_matmul(bf(2, 16), bf(1, 4, 16), i32(0, 2), x_scales=f32(2),
                                              w_scales=f32(1, 4))),
    (ValueError, lambda: vxmoe.grouped_matmul(f8(2, 16), f8(1, 4, 16), i32(0, 2))),
    (ValueError, lambda: vxmoe.grouped_matmul(f8(2, 16), f8(1, 4, 16), i32(0, 2), x_scales=f32(2))),
    (ValueError, lambda: vxmoe.grouped_matmul(f8(2, 16), f8(1, 4, 16), i32(0, 2), x_scales=f32(3),
                                              w_scales=f32(1, 4))),
    (TypeError, lambda: vxmoe.grouped_matmul(f8(2, 16), f8(1, 4, 16), i32(0, 2), x_scales=bf(2),
                                             w_scales=f32(1, 4))),
    (ValueError, lambda: vxmoe.grouped_matmul(f8(2, 24), f8(1, 4, 24), i32(0, 2), x_scales=f32(2),
                                              w_scales=f32(1, 4))),
    (TypeError, lambda: vxmoe.grouped_matmul(bf(2, 16), bf(1, 4, 16), i32(0, 2), out=f32(2, 4))),
    (ValueError, lambda: vxmoe.grouped_matmul(bf(2, 16), bf(1, 4, 16), i32(0, 2), out=bf(3, 4))),
    (ValueError, lambda: vxmoe.grouped_matmul(bf(2, 16), bf(1, 4, 16), i32(0, 2), out=bf(4, 2).t())),
    (ValueError, lambda: vxmoe.grouped_matmul(bf(2, 16), bf(1, 4, 16), i32(0, 2), out=bf(1, 4).expand(2, 4))),
    (TypeError, lambda: vxmoe.lora_add(bf(2, 8), f32(2, 16), bf(1, 8, 16), bf(1, 8, 8), i32(0, 0))),
    (TypeError, lambda: vxmoe.lora_add(bf(2, 8), bf(2, 16), f32(1, 8, 16), bf(1, 8, 8), i32(0, 0))),
    (TypeError, lambda: vxmoe.lora_add(bf(2, 8), bf(2, 16), bf(1, 8, 16), bf(1, 8, 8), f32(2))),
    (TypeError, lambda: vxmoe.lora_add(bf(2, 8), bf(2, 16), bf(1, 8, 16), bf(1, 8, 8), i32(0, 0), ranks=f32(1))),
    (ValueError, lambda: vxmoe.lora_add(bf(2, 8), bf(2, 16), bf(1, 12, 16), bf(1, 8, 12), i32(0, 0))),
    (ValueError, lambda: vxmoe.lora_add(bf(2, 8), bf(2, 16), bf(1, 264, 16), bf(1, 8, 264), i32(0, 0))),
    (ValueError, lambda: vxmoe.lora_add(bf(2, 8), bf(2, 12), bf(1, 8, 12), bf(1, 8, 8), i32(0, 0))),
    (ValueError, lambda: vxmoe.lora_add(bf(2, 8), bf(2, 16), bf(1, 8, 24), bf(1, 8, 8), i32(0, 0))),
    (ValueError, lambda: vxmoe.lora_add(bf(2, 8), bf(2, 16), bf(1, 8, 16), bf(1, 9, 8), i32(0, 0))),
    (ValueError, lambda: vxmoe.lora_add(bf(2, 8), bf(2, 16), bf(1, 8, 16), bf(2, 8, 8), i32(0, 0))),
    (ValueError, lambda: vxmoe.lora_add(bf(3, 8), bf(2, 16), bf(1, 8, 16), bf(1, 8, 8), i32(0, 0))),
    (ValueError, lambda: vxmoe.lora_add(bf(2, 8), bf(2, 16), bf(1, 8, 16), bf(1, 8, 8), i32(0, 0, 0))),
    (ValueError, lambda: vxmoe.lora_add(bf(2, 8), bf(2, 16), bf(1, 8, 16), bf(1, 8, 8), i32(0, 0), scales=f32(2))),
    (ValueError, lambda: vxmoe.lora_add(bf(2, 8), bf(2, 16), bf(1, 8, 16), bf(1, 8, 8), i32(0, 0), out=bf(2, 9))),
    (ValueError, lambda: vxmoe.lora_add(bf(2, 8), bf(2, 16), bf(1, 8, 16), bf(1, 8, 8), i32(0, 0),
                                        out=bf(8, 2).t())),
    (ValueError, lambda: vxmoe.lora_add(bf(2, 8), bf(2, 16), bf(129)[1:].view(1, 8, 16), bf(1, 8, 8), i32(0, 0))),
])
def test_refused(error, call):
    with pytest.raises(error):
        call()
