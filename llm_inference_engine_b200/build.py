"""Builds libmuse_proj.so (the sm_100a kernels + C ABI) in-tree with nvcc.

    python -m llm_inference_engine_b200.build [--force] [--verbose]

nvcc cross-compiles without a GPU. The library links the CUDA runtime statically and fetches the one
driver entry point it needs at run time, so it loads on a machine without a driver.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
# MUSE_TRACE=1 in the environment builds (and _capi loads) a separate diagnostic library whose kernels
# stamp their phases; the ordinary library carries none of that code.
TRACE = bool(os.environ.get("MUSE_TRACE"))
LIB_PATH = PKG_DIR / ("libmuse_proj_trace.so" if TRACE else "libmuse_proj.so")
SOURCES = ["gemv1.cu", "fewtok_mma.cu", "fewtok_zip.cu", "ffn_boundary.cu", "skinny_tc.cu", "gemm_tc.cu", "fp8_linear.cu", "fp8_gemm.cu", "rope_append.cu", "cache_attn.cu", "cache_attn_tc.cu", "capi.cu"]
# The torch-side binding of the 8-bit operators (a host-only extension module), beside the library.
BIND_SOURCE = CSRC / "bind.cpp"
NVCC_FLAGS = [
    "-std=c++17", "-O3", "-lineinfo",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-Xcompiler", "-fPIC", "--shared",
]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found: set NVCC or put /usr/local/cuda/bin on PATH")
    return cand


def _stale() -> bool:
    if not LIB_PATH.exists():
        return True
    built = LIB_PATH.stat().st_mtime
    deps = [CSRC / s for s in SOURCES] + list(CSRC.glob("*.cuh")) + [PKG_DIR.parent / "include" / "muse_proj.h"]
    return any(d.stat().st_mtime > built for d in deps)


def bind_path() -> Path:
    """Where the binding lies. It holds torch's and Python's C++ interfaces, which differ between their versions: the name says
    for which it was built, so that no other is ever loaded."""
    import sysconfig

    import torch

    return PKG_DIR / f"_bind.torch-{torch.__version__}{sysconfig.get_config_var('EXT_SUFFIX') or '.so'}"


def _bind_stale(path: Path) -> bool:
    deps = [BIND_SOURCE, PKG_DIR.parent / "include" / "muse_proj.h"]
    return not path.exists() or any(d.stat().st_mtime > path.stat().st_mtime for d in deps)


def build_bind(force: bool = False) -> Path:
    """Compile the binding if it is missing or older than its source; return its path."""
    path = bind_path()
    if not force and not _bind_stale(path):
        return path
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    nvcc = Path(_nvcc()).resolve()
    include = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", sysconfig.get_paths()["include"], nvcc.parent.parent / "include"]
    cmd = [shutil.which("g++") or "g++", "-std=c++17", "-O2", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-I{p}" for p in include], str(BIND_SOURCE), "-o", str(path), f"-L{root / 'lib'}", f"-Wl,-rpath,{root / 'lib'}",
           "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
        raise RuntimeError(f"g++ failed ({proc.returncode}) on {BIND_SOURCE.name}")
    return path


def _bind_or_say(make) -> None:
    """The binding is a shorter way to the library, not a part of it: where it cannot be built, calls go through Python."""
    try:
        make()
    except Exception as e:
        sys.stderr.write(f"the torch-side binding was not built ({e}): calls of the 8-bit operators go through Python\n")


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library and the binding where they are missing or older than their sources; return the library's path. A
    binding that cannot be built (no g++, no headers of Python or torch) is said, and the library built all the same."""
    if not force and not _stale():
        _bind_or_say(build_bind)
        return LIB_PATH
    nvcc = _nvcc()
    compile_flags = ([f for f in NVCC_FLAGS if f != "--shared"] + (["-Xptxas", "-v"] if verbose else [])
                     + (["-DMUSE_TRACE"] if TRACE else []))
    objs = [CSRC / (Path(s).stem + (".trace.o" if TRACE else ".o")) for s in SOURCES]

    def compile_one(src_obj):
        src, obj = src_obj
        return subprocess.run([nvcc, *compile_flags, "-c", str(CSRC / src), "-o", str(obj)], capture_output=True, text=True)

    from concurrent.futures import ThreadPoolExecutor

    with ThreadPoolExecutor(max_workers=len(SOURCES) + 1) as pool:   # one nvcc per translation unit, side by side
        bind = pool.submit(build_bind, force)
        results = list(pool.map(compile_one, zip(SOURCES, objs)))
    for src, proc in zip(SOURCES, results):
        if verbose or proc.returncode != 0:
            sys.stderr.write(proc.stdout + proc.stderr)
        if proc.returncode != 0:
            raise RuntimeError(f"nvcc failed ({proc.returncode}) on {src}")
    link = subprocess.run([nvcc, "--shared", "-Xcompiler", "-fPIC", "-gencode", "arch=compute_100a,code=sm_100a",
                           *[str(o) for o in objs], "-o", str(LIB_PATH)], capture_output=True, text=True)
    if link.returncode != 0:
        sys.stderr.write(link.stdout + link.stderr)
        raise RuntimeError(f"link failed ({link.returncode})")
    _bind_or_say(bind.result)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
