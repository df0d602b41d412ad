"""The attention half of the decode layer over an 8-bit cache: rotary positions and the append of new keys and values
(rope_append), and the attention that reads them (attention). They stand between the qkv_gate and the `o` projection;
attention_half() is that whole stretch.

Cache. A pool of pages of 64 tokens, held as e4m3 codes with one power-of-two scale per page and KV head (the number
format of fp8.py): K is [pages, heads, token, dim], V [pages, heads, dim, token] (transposed within the page: what the
attention's MMAs read without a transpose). A sequence owns the pages that its row of `page_table` names, page i holding its
tokens 64 i .. 64 i + 63. Pages may be shared for reading (a common prefix); the pages that a call appends to must belong
to one sequence of the batch each. A page's scale never shrinks while the page fills: when a new token raises it, the
codes of the page's earlier tokens are rounded to the new scale; writing a page's first token starts it afresh.

Batch. The new tokens of all sequences are the rows of one [m, ...] batch. cu_q [batch + 1] holds the first row of each
sequence, None means one new token per sequence. seq_lens counts the new tokens too: token j of a sequence's n new
ones has position seq_lens - n + j. A new token at a negative position (padding) is not appended, and its rows come back zero.

The calls read page_table, seq_lens and cu_q on the device, so they can be captured in a CUDA graph and replayed with
other lengths. What they find wrong there they report through check_status(): see its text.
"""

from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch

from . import _capi

PAGE = 64
HEAD_DIMS = (64, 128)
_INT_MAX = 0x7fffffff


class Cache8(NamedTuple):
    """The pool: k float8_e4m3fn [pages, heads, 64, dim], v float8_e4m3fn [pages, heads, dim, 64], and their exponent
    bytes uint8 [pages, heads] (a code stands for code * 2^(byte - 127)). All contiguous, on one device."""

    k: torch.Tensor
    v: torch.Tensor
    k_exp: torch.Tensor
    v_exp: torch.Tensor


def new_cache(pages: int, heads: int, dim: int, device) -> Cache8:
    """An empty pool."""
    if pages < 1 or heads < 1 or dim not in HEAD_DIMS:
        raise ValueError(f"a cache has at least one page and head of {HEAD_DIMS} dimensions, got pages={pages}, heads={heads}, dim={dim}")
    codes = lambda *shape: torch.zeros(shape, device=device, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scale = lambda: torch.full((pages, heads), 127, device=device, dtype=torch.uint8)
    return Cache8(codes(pages, heads, PAGE, dim), codes(pages, heads, dim, PAGE), scale(), scale())


def rotary_table(rot: int, positions: int, device, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 trained_positions: int | None = None) -> torch.Tensor:
    """cos and sin of every position's angles, FP32 [positions, rot / 2, 2], computed in FP64 once. Pair i of `rot`
    dimensions turns by position * base^(-2 i / rot). For contexts longer than the trained one:
      "linear"  positions are divided by `factor`
      "ntk"     base * factor^(rot / (rot - 2)): the slowest pair is slowed by `factor`, the fastest not at all
      "yarn"    pairs that make more than 32 turns over `trained_positions` keep their frequency, those that make less
                than one are slowed by `factor`, between them by a ramp that is linear in the number of turns; cos and sin
                grow by 0.1 ln(factor) + 1. (Many published models were trained with a ramp that is linear in the pair's
                index instead: their tables are to be made by the caller, in the same layout.)"""
    if rot < 2 or rot % 2 or positions < 1 or factor < 1.0:
        raise ValueError(f"rotary table of rot={rot} (even), positions={positions}, factor={factor} (at least 1)")
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    inv, amplitude = base ** (-2.0 * i / rot), 1.0
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "ntk":
        inv = (base * factor ** (rot / max(rot - 2, 1))) ** (-2.0 * i / rot)
    elif scaling == "yarn":
        if not trained_positions:
            raise ValueError('scaling "yarn" needs trained_positions')
        keep = ((trained_positions * inv / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        inv, amplitude = inv * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1.0
    elif scaling != "none":
        raise ValueError(f"unknown scaling {scaling!r}")
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return (amplitude * torch.stack([angle.cos(), angle.sin()], -1)).float().contiguous()


def check_status(device) -> None:
    """Wait for the device (all its streams) and raise if a call since the last check met a page index outside the pool (the
    page was neither read nor written), lengths or row bounds that do not fit the table, the batch or max_q (they were
    clamped), or gave up on a bounded wait. Not for use inside a stream capture. One word per device for the 8-bit operators,
    fp8's and all threads' among them: a check takes what any of them reported."""
    _capi.check_status_word(device)


_F8, _BF16, _U8, _I32 = torch.float8_e4m3fn, torch.bfloat16, torch.uint8, torch.int32


def _refuse_batch(cache: Cache8, page_table, seq_lens, cu_q, max_q: int, m: int, q_heads: int):
    """Says what is wrong with a batch that _check_batch() does not take."""
    k, v, ke, ve = cache
    dev = k.device
    if not k.is_cuda:
        raise RuntimeError(f"the cache is on {dev}: this path runs on a CUDA device only (no CPU fallback)")
    if k.dtype != _F8 or v.dtype != _F8 or ke.dtype != _U8 or ve.dtype != _U8:
        raise TypeError(f"a cache is float8_e4m3fn codes and uint8 exponents, got {k.dtype}, {v.dtype}, {ke.dtype}, {ve.dtype}")
    if k.dim() != 4 or k.shape[2] != PAGE or k.shape[3] not in HEAD_DIMS:
        raise ValueError(f"k must be [pages, heads, {PAGE}, dim] with dim in {HEAD_DIMS}, got {tuple(k.shape)}")
    pages, heads, _, dim = k.shape
    if v.shape != (pages, heads, dim, PAGE) or ke.shape != (pages, heads) or ve.shape != (pages, heads):
        raise ValueError(f"v {tuple(v.shape)} / exponents {tuple(ke.shape)}, {tuple(ve.shape)} do not fit k {tuple(k.shape)}")
    if not (k.is_contiguous() and v.is_contiguous() and ke.is_contiguous() and ve.is_contiguous()) or (k.data_ptr() | v.data_ptr()) % 16:
        raise ValueError("the cache's tensors must be contiguous and 16-byte aligned")
    if v.device != dev or ke.device != dev or ve.device != dev:
        raise ValueError("the cache's tensors must be on one device")
    if page_table.dim() != 2 or seq_lens.dim() != 1 or page_table.shape[0] != seq_lens.shape[0] or not seq_lens.shape[0] or not page_table.shape[1]:
        raise ValueError(f"page_table [batch, width] {tuple(page_table.shape)} and seq_lens [batch] {tuple(seq_lens.shape)} do not fit")
    batch = page_table.shape[0]
    for t in (page_table, seq_lens) if cu_q is None else (page_table, seq_lens, cu_q):
        if t.dtype != _I32 or not t.is_contiguous() or t.device != dev:
            raise TypeError("page_table, seq_lens and cu_q must be contiguous int32 tensors on the cache's device")
    if cu_q is None:
        if m != batch or max_q != 1:
            raise ValueError(f"without cu_q there is one new token per sequence: {m} rows for {batch} sequences, max_q={max_q}")
    elif cu_q.shape != (batch + 1,):
        raise ValueError(f"cu_q must be [batch + 1] = [{batch + 1}], got {tuple(cu_q.shape)}")
    raise ValueError(f"max_q={max_q} must be positive (and less than 2^31) and q_heads={q_heads} a multiple of the cache's {heads}")


def _check_batch(cache: Cache8, page_table, seq_lens, cu_q, max_q: int, m: int, q_heads: int):
    """The checks both operators share, in one expression; returns (device
    index, addresses of k, v, k_exp, v_exp, page_table, seq_lens, cu_q, pages, heads, dim, batch, width)."""
    k, v, ke, ve = cache
    shape, index = k.shape, k.get_device()
    if len(shape) == 4 and index >= 0:
        pages, heads, page, dim = shape
        kp, vp = k.data_ptr(), v.data_ptr()
        batch, width = page_table.shape if page_table.dim() == 2 else (0, 0)
        if (page == PAGE and (dim == 128 or dim == 64) and k.dtype is _F8 and v.dtype is _F8 and ke.dtype is _U8 and ve.dtype is _U8
                and v.shape == (pages, heads, dim, PAGE) and ke.shape == (pages, heads) and ve.shape == (pages, heads)
                and k.is_contiguous() and v.is_contiguous() and ke.is_contiguous() and ve.is_contiguous() and not (kp | vp) & 15
                and v.get_device() == index and ke.get_device() == index and ve.get_device() == index
                and batch and width and seq_lens.shape == (batch,) and page_table.dtype is _I32 and seq_lens.dtype is _I32
                and page_table.is_contiguous() and seq_lens.is_contiguous() and page_table.get_device() == index
                and seq_lens.get_device() == index and 1 <= max_q <= _INT_MAX and q_heads >= heads and not q_heads % heads):
            if cu_q is None:
                if m == batch and max_q == 1:
                    return index, kp, vp, ke.data_ptr(), ve.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(), None, pages, heads, dim, batch, width
            elif cu_q.shape == (batch + 1,) and cu_q.dtype is _I32 and cu_q.is_contiguous() and cu_q.get_device() == index:
                return (index, kp, vp, ke.data_ptr(), ve.data_ptr(), page_table.data_ptr(), seq_lens.data_ptr(), cu_q.data_ptr(), pages, heads, dim,
                        batch, width)
    _refuse_batch(cache, page_table, seq_lens, cu_q, max_q, m, q_heads)


def rope_append(qkv: torch.Tensor, cache: Cache8, cos_sin: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, *, q_heads: int,
                cu_q: torch.Tensor | None = None, max_q: int = 1, interleaved: bool = False, values: bool = False):
    """Turns q and k by their tokens' positions and appends k and v to the cache, one launch. qkv: BF16 [m, >= (q_heads +
    2 heads) dim], columns q | k | v (the rows of the qkv_gate projection as they are). cos_sin: rotary_table(rot, >= 64 *
    page_table.shape[1] positions), rot a multiple of 16 up to dim; pairs are (i, i + rot / 2), or neighbours when
    `interleaved`. max_q: at least the most new tokens of a sequence. Returns q BF16 [m, q_heads, dim]; with values=True
    (q, k, v), k and v BF16 [m, heads, dim]: the values that the cache then holds for the new tokens (for a prompt's own
    attention in 16 bits to see what later tokens will see)."""
    r = (_capi._BIND or _capi.bind()).rope_append(qkv, cache, cos_sin, page_table, seq_lens, cu_q, q_heads, max_q, interleaved, values)
    if r is not None:   # an ordinary call is done
        return r
    if qkv.dtype is not _BF16 or qkv.dim() != 2 or not qkv.shape[0]:
        raise TypeError(f"qkv must be BF16 [m, columns], got {qkv.dtype} {tuple(qkv.shape)}")
    m, width_in = qkv.shape
    index, kp, vp, kep, vep, tp, lp, cp, pages, heads, dim, batch, width = _check_batch(cache, page_table, seq_lens, cu_q, max_q, m, q_heads)
    cols = (q_heads + 2 * heads) * dim
    if qkv.get_device() != index or cos_sin.get_device() != index:
        raise ValueError("qkv and cos_sin must be on the cache's device")
    if width_in < cols:
        raise ValueError(f"qkv {tuple(qkv.shape)} is narrower than q | k | v = {cols} columns")
    if cos_sin.dtype is not torch.float32 or cos_sin.dim() != 3 or not cos_sin.is_contiguous() or cos_sin.data_ptr() & 15 or cos_sin.shape[2] != 2:
        raise TypeError(f"cos_sin must be a contiguous FP32 [positions, rot / 2, 2] table, got {cos_sin.dtype} {tuple(cos_sin.shape)}")
    positions, rot, _ = cos_sin.shape
    rot *= 2
    if rot % 16 or not 16 <= rot <= dim or positions < width * PAGE:
        raise ValueError(f"the table turns {rot} dimensions (a multiple of 16 up to {dim}) at {positions} positions; "
                         f"{width} pages per sequence need {width * PAGE}")
    ld, unit = qkv.stride()
    if unit != 1 or qkv.data_ptr() & 15 or (m > 1 and (ld & 7 or ld < width_in)):
        qkv = qkv[:, :cols].contiguous().clone()
        ld = cols
    dev = qkv.device
    with _capi.on_device(index):
        q = _capi.new_tensor((m, q_heads, dim), (q_heads * dim, dim, 1), _BF16, dev)
        k_val = v_val = kvp = vvp = None
        if values:
            k_val = _capi.new_tensor((m, heads, dim), (heads * dim, dim, 1), _BF16, dev)
            v_val = _capi.new_tensor((m, heads, dim), (heads * dim, dim, 1), _BF16, dev)
            kvp, vvp = k_val.data_ptr(), v_val.data_ptr()
        rc = _capi.load().muse_rope_append(qkv.data_ptr(), cos_sin.data_ptr(), tp, lp, cp, kp, vp, kep, vep, q.data_ptr(), kvp, vvp,
                                           _capi.status_ptr(index), ld if m > 1 else cols, m, batch, width, pages, max_q, q_heads, heads, dim,
                                           rot, 1 if interleaved else 0, min(positions, _INT_MAX), _capi.raw_stream(index))
    if rc:
        _capi.check(rc, f"muse_rope_append(m={m}, batch={batch}, q_heads={q_heads}, heads={heads}, dim={dim})")
    return (q, k_val, v_val) if values else q


def attention(q: torch.Tensor, cache: Cache8, page_table: torch.Tensor, seq_lens: torch.Tensor, *, cu_q: torch.Tensor | None = None,
              max_q: int = 1, scale: float | None = None, window: int = 0, gate: torch.Tensor | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q K^T) V over the cached tokens up to each query token's own position (the last `window` of them
    when window > 0), times sigmoid(gate) when gate is given: BF16 [m, q_heads * dim], ready for the `o` projection. A row
    that sees no token is zero; rows beyond the last sequence are left as they are. One call has one form, chosen by max_q times
    the query heads per KV head: up to 16 rows the cache is read at memory speed, above that in tiles of 128 rows whatever
    their filling, so sequences that decode single tokens are better not mixed with a prompt's chunk in one call (63 of 4000
    tokens beside a chunk of 512: 396 us, as two calls 182). q: BF16 [m, q_heads, dim]; gate: BF16
    [m, q_heads * dim] (the gate columns of qkv_gate, any row stride); scale: positive, 1 / sqrt(dim) by default; out
    (optional): BF16 [m, q_heads * dim] with unit column stride. Two launches, the same bits in every run."""
    if out is None:
        r = (_capi._BIND or _capi.bind()).attention(q, cache, page_table, seq_lens, cu_q, max_q, scale, window, gate)
        if r is not None:   # an ordinary call is done
            return r
    if q.dtype is not _BF16 or q.dim() != 3 or not q.shape[0]:
        raise TypeError(f"q must be BF16 [m, heads, dim], got {q.dtype} {tuple(q.shape)}")
    m, q_heads, d = q.shape
    index, kp, vp, kep, vep, tp, lp, cp, pages, heads, dim, batch, width = _check_batch(cache, page_table, seq_lens, cu_q, max_q, m, q_heads)
    max_q = min(max_q, m)   # no sequence has more new tokens than the batch has rows
    if d != dim or q.get_device() != index or window < 0:
        raise ValueError(f"q {tuple(q.shape)} on {q.device} does not fit the cache's heads of {dim}, or window={window} is negative")
    if scale is None:
        scale = 0.08838834764831845 if dim == 128 else 0.125
    elif not 0.0 < scale < math.inf:
        raise ValueError(f"scale={scale} must be positive")
    cols = q_heads * dim
    ld_q, head, unit = q.stride()
    if unit != 1 or head != dim or q.data_ptr() & 15 or (m > 1 and (ld_q & 7 or ld_q < cols)):
        q = q.contiguous().clone()
        ld_q = cols
    gp, ld_gate = None, 0
    if gate is not None:
        if gate.dtype is not _BF16 or gate.shape != (m, cols) or gate.get_device() != index:
            raise TypeError(f"gate must be BF16 [m, q_heads * dim] = [{m}, {cols}] on the cache's device, got {gate.dtype} {tuple(gate.shape)}")
        ld_gate, unit = gate.stride()
        if unit != 1 or (m > 1 and ld_gate < cols):
            gate = gate.contiguous().clone()
            ld_gate = cols
        gp = gate.data_ptr()
    ld_out = cols
    if out is not None:
        if out.dtype is not _BF16 or out.shape != (m, cols) or out.get_device() != index:
            raise TypeError(f"out must be BF16 [m, q_heads * dim] = [{m}, {cols}] on the cache's device, got {out.dtype} {tuple(out.shape)}")
        ld_out, unit = out.stride()
        if unit != 1 or (m > 1 and ld_out < cols):
            raise ValueError("out must have unit column stride and rows that do not overlap")
    dev = q.device
    with _capi.on_device(index):
        if out is None:
            out = _capi.new_tensor((m, cols), (cols, 1), _BF16, dev)
        # the workspace is the call's own (a captured graph keeps its own): calls may overlap on the GPU
        ws = _capi.new_tensor((_ws_bytes(index, batch, max_q, q_heads, heads, dim),), (1,), _U8, dev)
        rc = _capi.load().muse_cache_attention(q.data_ptr(), kp, vp, kep, vep, tp, lp, cp, gp, out.data_ptr(), ws.data_ptr(), _capi.status_ptr(index),
                                               ld_q if m > 1 else cols, ld_gate if m > 1 else cols, ld_out if m > 1 else cols, scale, m, batch,
                                               width, pages, max_q, q_heads, heads, dim, min(window, _INT_MAX), _capi.raw_stream(index))
    if rc:
        _capi.check(rc, f"muse_cache_attention(m={m}, batch={batch}, q_heads={q_heads}, heads={heads}, dim={dim})")
    return out


@functools.lru_cache(maxsize=4096)
def _ws_bytes(index: int, batch: int, max_q: int, q_heads: int, heads: int, dim: int) -> int:
    size = _capi.load().muse_cache_attention_ws_bytes(batch, max_q, q_heads, heads, dim)
    if size < 0:
        raise _capi.MuseError(f"muse_cache_attention_ws_bytes -> {size}")
    return size


def attention_half(data, state, cache: Cache8, cos_sin: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, *, q_heads: int,
                   cu_q: torch.Tensor | None = None, max_q: int = 1, window: int = 0, interleaved: bool = False, gated: bool = True,
                   eight_bit: bool = False) -> torch.Tensor:
    """The attention half of the decode layer: the qkv_gate projection, rope_append, attention, the `o` projection; its
    result is what muse_bf16_proj.attn_boundary takes as attn_out. data = {"x": BF16 [m, K]}; `state` as
    muse_bf16_proj.prepare made it, with "qkv_gate" (rows q | k | v | gate; without the gate rows when gated is False)
    and "o". eight_bit: both projections through kernel_fn_fp8 (prepare_fp8 made their 8-bit forms; the BF16 weights are not
    looked at). The rest as in rope_append and attention."""
    from . import muse_bf16_proj as proj

    project = proj.kernel_fn_fp8 if eight_bit else proj.kernel_fn
    x = data["x"]
    m = x.shape[0]
    heads, dim = cache.k.shape[1], cache.k.shape[3]
    qkv, cols = (q_heads + 2 * heads) * dim, q_heads * dim
    in_proj, out_proj = (proj.fp8_form(state, name)[0].shape if eight_bit else state[name].shape for name in ("qkv_gate", "o"))
    n, k = in_proj
    if n != qkv + (cols if gated else 0) or out_proj[1] != cols:
        raise ValueError(f"qkv_gate {tuple(in_proj)} and o {tuple(out_proj)} do not fit {q_heads} query heads and "
                         f"{heads} KV heads of {dim}, {'gated' if gated else 'not gated'}")
    rows = project({"x": x, "config": {"layer": "qkv_gate", "m": m, "n": n, "k": k}}, state)
    q = rope_append(rows, cache, cos_sin, page_table, seq_lens, q_heads=q_heads, cu_q=cu_q, max_q=max_q, interleaved=interleaved)
    a = attention(q, cache, page_table, seq_lens, cu_q=cu_q, max_q=max_q, window=window, gate=rows[:, qkv:] if gated else None)
    return project({"x": a, "config": {"layer": "o", "m": m, "n": out_proj[0], "k": cols}}, state)
