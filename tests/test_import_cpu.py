"""The package imports with a torch that was built without CUDA: the loader,
the prefill planner and the host combine need no device."""
from __future__ import annotations

import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_import_without_torch_cuda_bindings():
    program = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda")]:
    delattr(torch._C, name)
import vxmoe
x = torch.zeros((2, 64), dtype=torch.bfloat16)
for call in (lambda: vxmoe.add_rms_norm(x, None, x[0]), lambda: vxmoe.swiglu_e4m3(x, x),
             lambda: vxmoe.lora_add(x, x, x[None, :1].expand(1, 8, 64), x[None, :, :8], [0, 0])):
    try:
        call()
    except RuntimeError as e:
        assert "CUDA" in str(e)
    else:
        raise AssertionError("a CPU tensor was taken")
"""
    env = dict(os.environ, PYTHONPATH=os.path.join(ROOT, "veystrix-core_b200"))
    run = subprocess.run([sys.executable, "-c", program], env=env, capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stderr[-2000:]
