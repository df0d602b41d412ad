"""Projections with both operands in 8 bits: out = x @ W.T from e4m3 codes with a power-of-two scale per block.

An 8-bit value is an e4m3 code times 2^e. The exponent of a block whose largest finite magnitude is a is
e = max(ceil(log2(a / 448)), -64); it is held as the byte e + 127. Codes are rounded to nearest even, values that are not
finite become NaN. W has one exponent per 128 x 128 block, x one per token and 128 columns. Sums are FP32, the result is
BF16: the format costs a relative rounding of 2^-4 per code and nothing for the scale.

quantize_weight() makes the codes of a BF16 (or FP32) weight once; linear() is the product, quantising x on the way;
quantize() gives x's codes for callers that share them between several products. kernel_fn_fp8() of muse_bf16_proj is the
same behind the layer names of prepare().
"""

from __future__ import annotations

import functools

import torch

from . import _capi

BLOCK = 128
E_MIN = -64
_INT_MAX = 0x7fffffff
# What csrc/fp8_linear.cu takes in one launch; the rest csrc/fp8_gemm.cu (include/muse_proj.h has both sides' times).
WALK_MAX_TOKENS = 8
WALK_MAX_K = 8192
WALK_MAX_BYTES = 40 << 20


def _require(t: torch.Tensor, what: str, dtype: torch.dtype, dims: int) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{what} is on {t.device}: this path runs on a CUDA device only (no CPU fallback)")
    if t.dtype != dtype or t.dim() != dims:
        raise TypeError(f"{what} must be {dtype} with {dims} dimensions, got {t.dtype} {tuple(t.shape)}")


def exponent_byte(amax: torch.Tensor) -> torch.Tensor:
    """e + 127 of blocks with these largest magnitudes (int32): 448 = 0.875 * 2^9."""
    m, e = torch.frexp(amax.float())
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(min=E_MIN) + 127


def quantize_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """W [N, K] (BF16 or FP32, any device) as codes (float8_e4m3fn [N, K]) and exponent bytes (uint8
    [ceil(N / 128), ceil(K / 128)]). Done once; in torch."""
    if w.dim() != 2 or not w.is_floating_point():
        raise TypeError(f"a weight is a floating-point [N, K] tensor, got {w.dtype} {tuple(w.shape)}")
    n, k = w.shape
    f = w.float()
    a = torch.where(f.isfinite(), f.abs(), torch.zeros_like(f))
    a = torch.nn.functional.pad(a, (0, -k % BLOCK, 0, -n % BLOCK)).view(-(-n // BLOCK), BLOCK, -(-k // BLOCK), BLOCK).amax((1, 3))
    byte = exponent_byte(a)
    inv = ((254 - byte) << 23).to(torch.int32).view(torch.float32)
    y = (f * inv.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]).clamp(-448.0, 448.0)
    y = torch.where(f.isfinite(), y, torch.full_like(y, float("nan")))
    return y.to(torch.float8_e4m3fn).contiguous(), byte.to(torch.uint8).contiguous()


def dequantize_weight(w8: torch.Tensor, exponents: torch.Tensor) -> torch.Tensor:
    """The FP32 values that quantize_weight()'s codes stand for."""
    n, k = w8.shape
    scale = (exponents.to(torch.int32) << 23).view(torch.float32)
    return w8.float() * scale.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def _rows(x: torch.Tensor, m: int, k: int) -> torch.Tensor:
    """x itself where its rows can be read in 16-byte vectors (and their distance is an int), else a copy."""
    if x.stride(1) != 1 or x.data_ptr() % 16 or (m > 1 and (x.stride(0) % 8 or not k <= x.stride(0) <= _INT_MAX)):
        return x.contiguous().clone()
    return x


@functools.lru_cache(maxsize=4096)
def _ws_bytes(index: int, m: int, n: int, k: int) -> int:
    """Workspace of the many-token kernel's plan for a shape (the plan goes by sizes and the device's SM count)."""
    size = _capi.load().muse_fp8_gemm_ws_bytes(m, n, k)
    if size < 0:
        raise _capi.MuseError(f"muse_fp8_gemm_ws_bytes(m={m}, n={n}, k={k}) -> {size}")
    return size


def check_status(device) -> None:
    """Wait for the device (all its streams) and raise if a kernel since the last check gave up on one of its bounded waits. Not
    for use inside a stream capture. One word per device for the 8-bit operators, cache8's and all threads' among them: a
    check takes what any of them reported."""
    _capi.check_status_word(device)


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x BF16 [m, K], K a multiple of 16, as codes (float8_e4m3fn [m, K]) and exponent bytes (uint8 [m, ceil(K / 128)])."""
    _require(x, "x", torch.bfloat16, 2)
    m, k = x.shape
    if m < 1 or k < 16 or k % 16:
        raise ValueError(f"x must have at least one row and a multiple of 16 columns, got {tuple(x.shape)}")
    dev = x.device
    with _capi.on_device(dev.index):
        return _quantize(_rows(x, m, k), m, k, dev, dev.index)


def _quantize(x, m, k, dev, index):
    kb = -(-k // BLOCK)
    xq = _capi.new_tensor((m, k), (k, 1), torch.float8_e4m3fn, dev)
    xe = _capi.new_tensor((m, kb), (kb, 1), torch.uint8, dev)
    _capi.check(_capi.load().muse_fp8_quantize(x.data_ptr(), xq.data_ptr(), xe.data_ptr(), m, k, x.stride(0) if m > 1 else k,
                                               _capi.raw_stream(index)), "muse_fp8_quantize")
    return xq, xe


def _refuse_linear(x, w8, w_exp, out):
    """Says what is wrong with the arguments that linear() does not take."""
    if isinstance(x, (tuple, list)):
        xq, xe = x
        _require(xq, "x's codes", torch.float8_e4m3fn, 2)
        _require(xe, "x's exponents", torch.uint8, 2)
        m, k = xq.shape
        if xe.shape != (m, -(-k // BLOCK)) or not xq.is_contiguous() or not xe.is_contiguous() or xq.data_ptr() % 16:
            raise ValueError(f"x's codes {tuple(xq.shape)} and exponents {tuple(xe.shape)} must be contiguous, one exponent per 128 columns")
    else:
        _require(x, "x", torch.bfloat16, 2)
        m, k = x.shape
    _require(w8, "w8", torch.float8_e4m3fn, 2)
    _require(w_exp, "w_exp", torch.uint8, 2)
    n = w8.shape[0]
    if w8.shape[1] != k or m < 1 or n < 1 or k < 16 or k % 16:
        raise ValueError(f"x [{m}, {k}] and W {tuple(w8.shape)} do not fit, or K is not a multiple of 16")
    if w_exp.shape != (-(-n // BLOCK), -(-k // BLOCK)) or not w8.is_contiguous() or not w_exp.is_contiguous() or w8.data_ptr() % 16:
        raise ValueError(f"w8 {tuple(w8.shape)} and w_exp {tuple(w_exp.shape)} must be contiguous, one exponent per 128 x 128 block")
    if out is not None and (out.dtype != torch.bfloat16 or out.dim() != 2 or out.shape[0] != m or out.shape[1] < n or out.stride(1) != 1
                            or (m > 1 and not n <= out.stride(0) <= _INT_MAX)):
        raise ValueError("out must be BF16 [m, >= N] with unit column stride and rows less than 2^31 elements apart that do not overlap")
    raise ValueError("x, w8, w_exp and out must be on the same CUDA device")


_F8, _BF16, _U8 = torch.float8_e4m3fn, torch.bfloat16, torch.uint8


def linear(x, w8: torch.Tensor, w_exp: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """x @ W.T in BF16. `x`: BF16 [m, K] (any strides), or the pair that quantize() returns. `w8`, `w_exp`: the codes
    [N, K] and exponent bytes of W, contiguous; K a multiple of 16. `out` (optional): BF16 [m, >= N] with unit column
    stride, of which the first N columns are written. Weights are static: what made them must be complete before the first
    call (kernels may read them ahead of the work before them in the stream)."""
    if out is None:
        r = (_capi._BIND or _capi.bind()).linear(x, w8, w_exp)
        if r is not None:   # an ordinary call is done
            return r
    # One expression takes what is right; what it does not take is looked at again to say why.
    pair = isinstance(x, (tuple, list))
    xt = x[0] if pair else x
    shape, w_shape, index = xt.shape, w8.shape, w8.get_device()
    if len(shape) != 2 or len(w_shape) != 2:
        _refuse_linear(x, w8, w_exp, out)
    m, k = shape
    n = w_shape[0]
    kb = (k + 127) // 128
    if not (m >= 1 and n >= 1 and k >= 16 and not k & 15 and w_shape[1] == k and index >= 0 and xt.get_device() == index
            and w_exp.get_device() == index and w8.dtype is _F8 and w_exp.dtype is _U8 and w_exp.shape == ((n + 127) // 128, kb)
            and w8.is_contiguous() and w_exp.is_contiguous() and not w8.data_ptr() & 15
            and (xt.dtype is _BF16 if not pair else
                 xt.dtype is _F8 and x[1].dtype is _U8 and x[1].shape == (m, kb) and xt.is_contiguous() and x[1].is_contiguous()
                 and x[1].get_device() == index and not xt.data_ptr() & 15)):
        _refuse_linear(x, w8, w_exp, out)
    ld_out = n
    if out is not None:
        if (out.dtype is not _BF16 or out.dim() != 2 or out.shape[0] != m or out.shape[1] < n or out.get_device() != index or out.stride(1) != 1
                or (m > 1 and not n <= out.stride(0) <= _INT_MAX)):
            _refuse_linear(x, w8, w_exp, out)
        if m > 1:
            ld_out = out.stride(0)
    lib, dev = _capi.load(), w8.device
    with _capi.on_device(index):
        if out is None:
            out = _capi.new_tensor((m, n), (n, 1), _BF16, dev)
        if not pair:
            x = _rows(x, m, k)
            if m <= WALK_MAX_TOKENS and k <= WALK_MAX_K and n * k <= WALK_MAX_BYTES:
                rc = lib.muse_fp8_walk(w8.data_ptr(), w_exp.data_ptr(), x.data_ptr(), out.data_ptr(), m, n, k, x.stride(0) if m > 1 else k, ld_out,
                                       _capi.raw_stream(index))
                if rc:
                    _capi.check(rc, f"muse_fp8_walk(m={m}, n={n}, k={k})")
                return out
            xq, xe = _quantize(x, m, k, dev, index)
        else:
            xq, xe = x
        size = _ws_bytes(index, m, n, k)
        ws = _capi.new_tensor((size,), (1,), _U8, dev) if size else None   # the call's own: calls may overlap on the GPU
        rc = lib.muse_fp8_gemm(w8.data_ptr(), w_exp.data_ptr(), xq.data_ptr(), xe.data_ptr(), out.data_ptr(), ws.data_ptr() if size else None,
                               _capi.status_ptr(index), m, n, k, ld_out, _capi.raw_stream(index))
    if rc:
        _capi.check(rc, f"muse_fp8_gemm(m={m}, n={n}, k={k})")
    return out
