"""The 8-bit operators without a GPU: the weight codes and the rotary tables that the host makes, and what the Python
functions and the C entries refuse before anything is launched."""

from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

from llm_inference_engine_b200 import cache8, fp8


def weight(n, k, seed, scale=0.02):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, k, generator=g) * scale).bfloat16()


@pytest.mark.parametrize("n,k", [(1, 16), (128, 128), (129, 144), (300, 400)])
def test_weight_codes_are_within_half_a_step(n, k):
    w = weight(n, k, 5 + n)
    w[0, 0] = 3.0   # one block with another scale
    codes, exps = fp8.quantize_weight(w)
    assert codes.shape == (n, k) and exps.shape == (-(-n // 128), -(-k // 128))
    back = fp8.dequantize_weight(codes, exps).double()
    step = torch.exp2(exps.double() - 127).repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    # e4m3: 2^-4 of a normal value, half of the subnormals' step 2^-9 below 2^-6
    bound = torch.maximum(w.double().abs() * 2.0**-4, step * 2.0**-10)
    assert bool(((back - w.double()).abs() <= bound).all())
    for i in range(exps.shape[0]):   # the smallest exponent that holds the block's largest value
        for j in range(exps.shape[1]):
            a = w[128 * i : 128 * i + 128, 128 * j : 128 * j + 128].double().abs().max().item()
            e = int(exps[i, j]) - 127
            assert a <= 448.0 * 2.0**e and (a > 448.0 * 2.0 ** (e - 1) or e == fp8.E_MIN)


def test_weight_exponents_at_their_borders():
    for a, e in ((448.0, 0), (450.0, 1), (224.0, -1), (0.0, fp8.E_MIN), (2.0**-100, fp8.E_MIN), (1.75 * 2.0**127, 119)):
        assert int(fp8.exponent_byte(torch.tensor(a))) == e + 127, a
    w = torch.zeros(2, 16)
    w[0, 0], w[0, 1], w[1, 0] = math.inf, math.nan, 1.0   # what is not finite has no part in the scale
    codes, exps = fp8.quantize_weight(w)
    back = fp8.dequantize_weight(codes, exps)
    assert torch.isnan(back[0, :2]).all() and back[1, 0] == 1.0 and int(exps) == 127 - 8


@pytest.mark.parametrize("scaling,factor,trained", [("none", 1.0, None), ("linear", 4.0, None), ("ntk", 2.0, None), ("yarn", 8.0, 2048)])
def test_rotary_table(scaling, factor, trained):
    rot, base = 64, 10000.0
    table = cache8.rotary_table(rot, 500, "cpu", base=base, scaling=scaling, factor=factor, trained_positions=trained)
    assert table.shape == (500, rot // 2, 2) and table.dtype == torch.float32
    for i in (0, 5, 17, 31):
        inv, amp = base ** (-2 * i / rot), 1.0
        if scaling == "linear":
            inv /= factor
        elif scaling == "ntk":
            inv = (base * factor ** (rot / (rot - 2))) ** (-2 * i / rot)
        elif scaling == "yarn":
            keep = min(max((trained * inv / (2 * math.pi) - 1) / 31, 0), 1)
            inv, amp = inv * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1
        for p in (0, 1, 499):
            # rounded once: half a step of values below 2
            assert abs(table[p, i, 0].item() - amp * math.cos(p * inv)) <= 2.0**-23
            assert abs(table[p, i, 1].item() - amp * math.sin(p * inv)) <= 2.0**-23
    for bad in (dict(rot=3), dict(rot=0), dict(positions=0), dict(factor=0.5), dict(scaling="other"), dict(scaling="yarn", trained_positions=None)):
        args = dict(rot=64, positions=4, device="cpu", scaling="none", factor=1.0)
        args.update(bad)
        with pytest.raises(ValueError):
            cache8.rotary_table(**args)


def test_cpu_tensors_are_refused():
    w8, we = fp8.quantize_weight(weight(128, 128, 1))
    x = weight(4, 128, 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fp8.linear(x, w8, we)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fp8.quantize(x)
    with pytest.raises(TypeError):
        fp8.quantize_weight(torch.zeros(4, 4, dtype=torch.int32))
    cache = cache8.new_cache(2, 2, 64, "cpu")
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cache8.attention(torch.zeros(1, 4, 64, dtype=torch.bfloat16), cache, table, lens)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cache8.rope_append(torch.zeros(1, 512, dtype=torch.bfloat16), cache, cache8.rotary_table(64, 128, "cpu"), table, lens, q_heads=4)
    for bad in (dict(pages=0), dict(heads=0), dict(dim=96)):
        args = dict(pages=2, heads=2, dim=64, device="cpu")
        args.update(bad)
        with pytest.raises(ValueError):
            cache8.new_cache(**args)


# The C entries: an argument that is wrong comes back as a negative code before any pointer is followed or anything launched.
# P stands for addresses that are aligned and never read.
P, ODD = 1 << 20, (1 << 20) + 2

QUANTIZE = dict(x=P, xq=P, xe=P, m=4, K=128, ld_x=128, stream=None)
WALK = dict(W=P, we=P, x=P, out=P, m=4, N=128, K=128, ld_x=128, ld_out=128, stream=None)
GEMM = dict(W=P, we=P, xq=P, xe=P, out=P, ws=None, status=P, m=40, N=128, K=128, ld_out=128, stream=None)
ROPE = dict(qkv=P, cos_sin=P, page_table=P, seq_lens=P, cu_q=P, k=P, v=P, k_exp=P, v_exp=P, q_out=P, k_val=P, v_val=P, status=P, ld_qkv=1024, m=4, batch=2,
            width=3, pages=9, max_q=3, hq=4, hk=2, dim=128, rot=64, interleaved=0, table_rows=192, stream=None)
ATTEND = dict(q=P, k=P, v=P, k_exp=P, v_exp=P, page_table=P, seq_lens=P, cu_q=P, gate=P, out=P, ws=P, status=P, ld_q=512, ld_gate=512, ld_out=512, scale=0.1,
              m=4, batch=2, width=3, pages=9, max_q=3, hq=4, hk=2, dim=128, window=0, stream=None)
REFUSED = (
    [("muse_fp8_quantize", QUANTIZE, dict(bad)) for bad in ([("x", None)], [("xq", None)], [("xe", None)], [("m", 0)], [("K", 120)], [("K", 0)], [("ld_x", 120)],
                                                            [("ld_x", 132)], [("x", ODD)], [("xq", ODD)])]
    + [("muse_fp8_walk", WALK, dict(bad)) for bad in ([("W", None)], [("we", None)], [("x", None)], [("out", None)], [("m", 9)], [("m", 0)], [("N", 0)], [("K", 24)],
                                                      [("K", 8208), ("ld_x", 8208)], [("ld_x", 64)], [("ld_x", 130)], [("ld_out", 64)], [("W", ODD)], [("x", ODD)])]
    + [("muse_fp8_gemm", GEMM, dict(bad)) for bad in ([("W", None)], [("we", None)], [("xq", None)], [("xe", None)], [("out", None)], [("status", None)], [("m", 0)],
                                                      [("N", 0)], [("K", 100)], [("ld_out", 127)], [("W", ODD)], [("xq", ODD)])]
    + [("muse_rope_append", ROPE, dict(bad)) for bad in ([("qkv", None)], [("cos_sin", None)], [("page_table", None)], [("seq_lens", None)], [("k", None)], [("v_exp", None)],
                                                         [("q_out", None)], [("status", None)], [("k_val", None)], [("v_val", None)], [("cu_q", None)],
                                                         [("cu_q", None), ("max_q", 1)], [("m", 0)], [("batch", 0)], [("width", 0)], [("width", 1 << 26)], [("pages", 0)],
                                                         [("max_q", 0)], [("hk", 0)], [("dim", 96)], [("rot", 8)], [("rot", 72)], [("rot", 144)], [("table_rows", 191)],
                                                         [("ld_qkv", 1016)], [("ld_qkv", 1028)], [("hk", 0x7fffffff)], [("qkv", ODD)], [("k", ODD)], [("v_val", ODD)])]
    + [("muse_cache_attention", ATTEND, dict(bad)) for bad in ([("q", None)], [("k", None)], [("v_exp", None)], [("page_table", None)], [("out", None)], [("ws", None)],
                                                               [("status", None)], [("cu_q", None)], [("cu_q", None), ("max_q", 1)], [("m", 0)], [("batch", 0)],
                                                               [("width", 0)], [("width", 1 << 26)], [("pages", 0)], [("max_q", 0)], [("max_q", 1 << 30)], [("hk", 3)],
                                                               [("hq", 1)], [("dim", 32)], [("window", -1)], [("ld_q", 508)], [("ld_q", 504)], [("ld_gate", 511)],
                                                               [("ld_out", 511)], [("scale", 0.0)], [("scale", -1.0)], [("scale", math.inf)], [("scale", math.nan)],
                                                               [("q", ODD)], [("v", ODD)], [("ws", ODD)], [("out", P + 1)], [("gate", P + 1)])]
)


@pytest.mark.parametrize("name,good,bad", REFUSED, ids=[f"{n[5:]}-{'-'.join(f'{k}={v}' for k, v in b.items())}" for n, _, b in REFUSED])
def test_c_entries_refuse(name, good, bad):
    from llm_inference_engine_b200 import _capi

    assert _call(getattr(_capi.load(), name), good, bad) < 0


def _call(fn, good, bad):
    args = dict(good)
    args.update(bad)
    return fn(*[C.c_float(v) if k == "scale" else v for k, v in args.items()])


def test_workspace_sizes_are_refused_or_positive_without_arguments_to_match():
    from llm_inference_engine_b200 import _capi

    lib = _capi.load()
    for args in ((0, 128, 128), (4, 0, 128), (4, 128, 100)):
        assert lib.muse_fp8_gemm_ws_bytes(*args) < 0
    for args in ((0, 1, 4, 2, 128), (1, 0, 4, 2, 128), (1, 1, 4, 3, 128), (1, 1, 1, 2, 128), (1, 1, 4, 2, 96)):
        assert lib.muse_cache_attention_ws_bytes(*args) < 0
