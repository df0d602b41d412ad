"""What a machine with less than the usual set of tools or builds still gets. No GPU."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch

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


class Tools:
    """subprocess.run of the build: nvcc works, g++ is missing or fails."""

    def __init__(self, missing):
        self.missing, self.ran = missing, []

    def __call__(self, cmd, **kw):
        self.ran.append(cmd)
        if "bind.cpp" in " ".join(cmd):
            if self.missing:
                raise FileNotFoundError(cmd[0])
            return subprocess.CompletedProcess(cmd, 1, "", "Python.h: No such file or directory")
        return subprocess.CompletedProcess(cmd, 0, "", "")


@pytest.mark.parametrize("missing", [True, False])
@pytest.mark.parametrize("force", [True, False])
def test_the_library_is_built_without_the_binding(monkeypatch, tmp_path, capfd, missing, force):
    from llm_inference_engine_b200 import build

    tools = Tools(missing)
    monkeypatch.setattr(build.subprocess, "run", tools)
    monkeypatch.setattr(build, "LIB_PATH", tmp_path / "lib.so")
    monkeypatch.setattr(build, "bind_path", lambda: tmp_path / "bind.so")
    assert build.build(force=force) == tmp_path / "lib.so"
    links = [cmd for cmd in tools.ran if str(tmp_path / "lib.so") in cmd]
    assert len(links) == 1 and sum("-c" in cmd for cmd in tools.ran) == len(build.SOURCES)
    assert "binding was not built" in capfd.readouterr().err


def test_calls_go_through_python_without_the_binding(monkeypatch, tmp_path):
    from llm_inference_engine_b200 import _capi, build, fp8

    monkeypatch.setattr(build.subprocess, "run", Tools(False))
    monkeypatch.setattr(build, "bind_path", lambda: tmp_path / "bind.so")
    monkeypatch.setattr(_capi, "_BIND", None)
    with pytest.warns(RuntimeWarning, match="go through Python"):
        assert _capi.bind().linear(None, None, None) is None
    w8, we = fp8.quantize_weight(torch.ones(16, 16))
    with pytest.raises(RuntimeError, match="no CPU fallback"):   # what the Python way says
        fp8.linear(torch.ones(1, 16, dtype=torch.bfloat16), w8, we)


def test_a_binding_of_another_torch_is_not_taken(monkeypatch):
    """What was built against one torch stays beside what is built against another, and neither is loaded for the other."""
    from llm_inference_engine_b200 import _capi, build

    here = build.build_bind()
    assert here.exists() and here == build.bind_path()
    monkeypatch.setattr(torch, "__version__", "9.9.9+other")
    tools = Tools(False)
    monkeypatch.setattr(build.subprocess, "run", tools)
    assert build.bind_path() != here and not build.bind_path().exists()
    monkeypatch.setattr(_capi, "_BIND", None)
    with pytest.warns(RuntimeWarning):
        _capi.bind()
    assert len(tools.ran) == 1 and str(build.bind_path()) in tools.ran[0]   # it tried to build its own
