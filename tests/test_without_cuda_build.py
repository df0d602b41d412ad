"""What a machine with less than the usual set of tools or builds still gets. No GPU."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_the_package_imports_on_a_torch_without_cuda():
    """Such a torch lacks the functions of torch._C that read the current device and stream."""
    program = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_get")]:
    delattr(torch._C, name)
from llm_inference_engine_b200 import _capi, cache8, fp8, muse_bf16_proj, plan, tp, zip12
codes, exps = fp8.quantize_weight(torch.ones(4, 16))
assert bool((fp8.dequantize_weight(codes, exps) == 1).all())
cache8.rotary_table(64, 4, "cpu")
"""
    done = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
