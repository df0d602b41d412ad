"""ctypes binding of libmuse_proj.so (declarations: include/muse_proj.h).

The library is the only compute path: if it is missing and cannot be built, loading raises and so
does every call that needs it. There is no PyTorch or CPU fallback.
"""

from __future__ import annotations

import ctypes as C
import threading
import warnings
from pathlib import Path

import torch

from . import build as _build

_LIB = None

# name -> (restype, argtypes); kept in one place so that the symbol-export test can walk it.
SIGNATURES = {
    "muse_abi_version": (C.c_int, []),
    "muse_set_programmatic_launch": (C.c_int, [C.c_int]),
    "muse_query": (C.c_int, [C.c_int]),
    "muse_gemv1": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int,
                             C.c_void_p, C.c_void_p, C.c_void_p]),
    "muse_tmap_encode_2d": (C.c_int, [C.c_void_p, C.c_void_p, C.c_longlong, C.c_longlong, C.c_longlong, C.c_int]),
    "muse_skinny_ws_floats": (C.c_longlong, [C.c_int, C.c_int, C.c_int]),
    "muse_skinny_tiles": (C.c_int, [C.c_int, C.c_int, C.c_int]),
    "muse_skinny_stage_bytes": (C.c_int, [C.c_int, C.c_int]),
    "muse_skinny_tc": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                 C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int,
                                 C.c_void_p, C.c_void_p]),
    "muse_skinny_smem_bytes": (C.c_int, [C.c_int, C.c_int, C.c_int, C.c_int, C.c_int]),
    "muse_skinny_max_clusters": (C.c_int, [C.c_int, C.c_int, C.c_int, C.c_int, C.c_int]),
    "muse_nop": (C.c_int, [C.c_void_p]),
    "muse_copy_h2d_async": (C.c_int, [C.c_void_p, C.c_void_p, C.c_longlong, C.c_void_p]),
    "muse_copy_d2h_sync": (C.c_int, [C.c_void_p, C.c_void_p, C.c_longlong, C.c_void_p]),
    "muse_fetch_host": (C.c_int, [C.c_void_p, C.c_void_p, C.c_longlong, C.c_void_p]),
    "muse_fewtok_mma_host": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int,
                                       C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p]),
    "muse_fewtok_mma": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int,
                                  C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]),
    "muse_fewtok_rowpar": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int,
                                     C.c_void_p, C.c_void_p, C.c_void_p]),
    "muse_fewtok_smem_bytes": (C.c_longlong, [C.c_int, C.c_int, C.c_int]),
    "muse_fewtok_f32": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int,
                                  C.c_int, C.c_int, C.c_void_p]),
    "muse_attn_boundary": (C.c_int, [C.c_void_p, C.c_int, C.c_int, C.c_void_p]),
    "muse_fewtok_boundary": (C.c_int, [C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int,
                                       C.c_void_p, C.c_void_p]),
    "muse_boundary_pooler_router": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                              C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p, C.c_void_p,
                                              C.c_void_p]),
    "muse_fewtok_zip": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_int, C.c_int,
                                  C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p]),
    "muse_ffn_boundary": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_void_p]),
    "muse_unpooler_ffn_boundary": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int,
                                             C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]),
    "muse_gemm_tc_smem_bytes": (C.c_int, [C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int]),
    "muse_gemm_tc_max_clusters": (C.c_int, [C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int]),
    "muse_gemm_tc_ws_floats": (C.c_longlong, [C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int]),
    "muse_gemm_tc_cnt_ints": (C.c_int, [C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int]),
    "muse_gemm_tc": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int,
                               C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int,
                               C.c_void_p, C.c_void_p]),
    "muse_static_scratch_floats": (C.c_longlong, []),
    "muse_static_scratch_tiles": (C.c_int, []),
    "muse_skinny_tc_noalloc": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int,
                                         C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int,
                                         C.c_void_p]),
    "muse_fp8_quantize": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_void_p]),
    "muse_fp8_walk": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p]),
    "muse_fp8_gemm_ws_bytes": (C.c_longlong, [C.c_int] * 3),
    "muse_fp8_gemm": (C.c_int, [C.c_void_p] * 7 + [C.c_int] * 4 + [C.c_void_p]),
    "muse_rope_append": (C.c_int, [C.c_void_p] * 13 + [C.c_longlong] + [C.c_int] * 11 + [C.c_void_p]),
    "muse_cache_attention_ws_bytes": (C.c_longlong, [C.c_int] * 5),
    "muse_cache_attention": (C.c_int, [C.c_void_p] * 12 + [C.c_longlong] * 3 + [C.c_float] + [C.c_int] * 9 + [C.c_void_p]),
    "muse_cache_attention_plan": (C.c_longlong, [C.c_void_p] * 2 + [C.c_int] * 8 + [C.c_void_p, C.c_longlong]),
    "muse_cache_attention_join": (C.c_longlong, [C.c_void_p] * 2 + [C.c_int] * 10 + [C.c_void_p, C.c_longlong]),
}

ABI_VERSION = 19


class MuseError(RuntimeError):
    """A C-ABI call returned non-zero (negative: rejected argument; positive: CUDA error)."""


def lib_path() -> Path:
    return _build.LIB_PATH


def load(build_if_missing: bool = True):
    """Load (building first if needed) and type the library. Raises if that is impossible."""
    global _LIB
    if _LIB is not None:
        return _LIB
    path = lib_path()
    if not path.exists():
        if not build_if_missing:
            raise MuseError(f"{path} is missing: run `python -m llm_inference_engine_b200.build`")
        _build.build()
    lib = C.CDLL(str(path))
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)  # AttributeError here = the library does not export the symbol
        fn.restype = res
        fn.argtypes = args
    if lib.muse_abi_version() != ABI_VERSION:
        raise MuseError(f"{path}: ABI {lib.muse_abi_version()} != expected {ABI_VERSION}; rebuild")
    _LIB = lib
    return lib


_BIND = None


class _NoBinding:
    """In the binding's place where it cannot be built: no call is an ordinary one."""

    linear = rope_append = attention = staticmethod(lambda *args: None)
    set_status = staticmethod(lambda index, address: None)


def bind():
    """The torch-side binding of the 8-bit operators (csrc/bind.cpp): their ordinary calls in one step. Built with the
    library. Where it is missing and cannot be built, every call takes the way through Python to the same entry points (10 us
    of host time more), and a warning says so once."""
    global _BIND
    if _BIND is None:
        from importlib.machinery import ExtensionFileLoader
        from importlib.util import module_from_spec, spec_from_loader

        lib = load()
        try:
            path = _build.bind_path()
            path = str(path if path.exists() else _build.build_bind())
        except Exception as e:
            warnings.warn(f"the torch-side binding cannot be built ({e}): calls of the 8-bit operators go through Python", RuntimeWarning, stacklevel=2)
            _BIND = _NoBinding
            return _BIND
        loader = ExtensionFileLoader("_bind", path)
        module = module_from_spec(spec_from_loader("_bind", loader))
        loader.exec_module(module)
        module.set_entries(*[C.cast(getattr(lib, f"muse_{name}"), C.c_void_p).value
                             for name in ("fp8_walk", "fp8_quantize", "fp8_gemm", "fp8_gemm_ws_bytes", "rope_append", "cache_attention",
                                          "cache_attention_ws_bytes")])
        for index, word in _STATUS.items():
            module.set_status(index, word.data_ptr())
        _BIND = module
    return _BIND


def check(rc: int, what: str) -> None:
    if rc != 0:
        kind = "rejected argument" if rc < 0 else "CUDA error"
        raise MuseError(f"{what}: {kind} {rc}")


# Small calls are bound by what the host does for them: the two helpers below are torch.cuda.current_stream(i).cuda_stream
# and torch.cuda.device(i) without the objects those build (2 us and 1 us a call). A torch without CUDA has neither; the host
# side of the package works with it all the same.
raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class on_device:
    """torch.cuda.device for the calls that nearly always find their device current."""

    __slots__ = ("index", "was")

    def __init__(self, index: int):
        self.index = index

    def __enter__(self):
        self.was = _current_device()
        if self.was != self.index:
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.was != self.index:
            torch.cuda.set_device(self.was)


def new_tensor(shape, strides, dtype, device) -> torch.Tensor:
    """torch.empty of known strides (1.5 us against 2.3)."""
    return torch.empty_strided(shape, strides, dtype=dtype, device=device)


_STATUS: dict[int, torch.Tensor] = {}
_STATUS_LOCK = threading.Lock()
STATUS_TEXT = ((128, "a page index outside the pool"), (256, "lengths or row bounds that do not fit"))


def status_ptr(index: int) -> int:
    """Address of the status word that the 8-bit operators of a device share (the projections of prepare() have one per
    state)."""
    word = _STATUS.get(index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():   # it must outlive the graph
            raise MuseError("the first call of the 8-bit operators on a device makes their status word: make it outside stream capture")
        with _STATUS_LOCK:   # one word per device, whoever comes first
            word = _STATUS.get(index)
            if word is None:
                word = torch.zeros(1, device=torch.device("cuda", index), dtype=torch.int32)
                torch.cuda.synchronize(word.device)   # a report from another stream must not meet the filling with zero
                _STATUS[index] = word
                bind().set_status(index, word.data_ptr())
    return word.data_ptr()


def check_status_word(device) -> None:
    """Waits for the whole device, whatever stream the calls ran on, and raises what they have reported; takes away the bits it
    raises and no others."""
    device = torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    word = _STATUS.get(index)
    if word is None:
        return
    torch.cuda.synchronize(torch.device("cuda", index))
    bits = int(word.item())
    if bits:
        word.bitwise_and_(~bits)
        what = [text for bit, text in STATUS_TEXT if bits & bit] + (["a timed-out wait"] if bits & ~384 else [])
        raise MuseError(f"the 8-bit operators reported: {', '.join(what)} (status bits {bits:#x}, see MUSE_ST_* in muse_proj.h)")


MAX_WORLD = 8
LL_TOKENS = 32   # MUSE_LL_TOKENS: most tokens of a column-parallel muse_fewtok_mma call
RP_TOKENS = 8    # MUSE_RP_TOKENS: most tokens of a row-parallel muse_fewtok_rowpar call


class PeerSync(C.Structure):
    """muse_peer_sync_t: where a column-parallel kernel writes its slice on every rank (muse_proj.h)."""

    _fields_ = [("world", C.c_int), ("rank", C.c_int), ("col0", C.c_int), ("reserved", C.c_int),
                ("out", C.c_void_p * MAX_WORLD), ("flags", C.c_void_p * MAX_WORLD), ("ll", C.c_void_p * MAX_WORLD)]


class Boundary(C.Structure):
    """muse_boundary_t: the operands of the post-attention boundary (muse_proj.h)."""

    _fields_ = [("stream", C.c_void_p), ("attn_out", C.c_void_p), ("alpha", C.c_void_p), ("beta", C.c_void_p),
                ("norm_w", C.c_void_p), ("stream1", C.c_void_p), ("h", C.c_void_p), ("h_f32", C.c_void_p)]


class FfnBoundary(C.Structure):
    """muse_ffn_boundary_t: the operands of the post-FFN boundary (muse_proj.h)."""

    _fields_ = [("stream1", C.c_void_p), ("alpha", C.c_void_p), ("beta", C.c_void_p), ("post_w", C.c_void_p),
                ("next_w", C.c_void_p), ("stream2", C.c_void_p), ("hidden", C.c_void_p)]


class TensorMap:
    """A 128-byte CUtensorMap blob in host memory, 64-byte aligned as the driver requires."""

    def __init__(self):
        self._raw = C.create_string_buffer(128 + 64)
        base = C.addressof(self._raw)
        self.ptr = (base + 63) & ~63

    @classmethod
    def for_matrix(cls, data_ptr: int, rows: int, cols: int, row_stride_bytes: int, box_rows: int) -> "TensorMap":
        tm = cls()
        check(load().muse_tmap_encode_2d(tm.ptr, data_ptr, rows, cols, row_stride_bytes, box_rows),
              f"muse_tmap_encode_2d(rows={rows}, cols={cols}, box_rows={box_rows})")
        return tm
