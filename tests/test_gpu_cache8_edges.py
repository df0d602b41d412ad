"""The attention over the 8-bit cache where factors and weights leave the middle of their ranges, against 64 bits. Tolerances as in
test_gpu_cache8.py unless a test says otherwise. Each case runs with 8, 16 and 128 rows per KV head (the kernels' tiles)."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_cache8 import DEV, PAGE, attention64, bounds, filled_cache, i32, make_table

pytestmark = pytest.mark.gpu
HEADS = [(2, 8), (1, 16), (1, 128)]   # new tokens of a sequence and rows per KV head: 2 x 4, 1 x 16, 1 x 128


@pytest.fixture(scope="module")
def c8():
    from llm_inference_engine_b200 import cache8

    return cache8


@pytest.mark.parametrize("new,rows", HEADS)
@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("size", [0.0, 2.0**-95, 2.0**120])
def test_queries_of_any_size_over_pages_of_zero_keys(c8, new, rows, window, size):
    """Keys of zero are kept under the smallest exponent (byte 63): every score is zero and the result the mean of the seen v.
    The queries' own power of two times that of the page leaves FP32's range downward when the row is zero or tiny."""
    hk, dim = 2, 64
    hq = hk * rows // new
    lens = [1 if new == 1 else 2, 63, 150, 64]
    m, cu = 4 * new, bounds([new] * 4)
    need = sum(-(-n // PAGE) for n in lens)
    cache = filled_cache(c8, need + 1, hk, dim, 5 + rows)
    cache.k.view(torch.uint8).zero_()
    cache.k_exp.fill_(63)
    table = make_table(lens, 4, need + 1, rows)
    g = torch.Generator(device=DEV).manual_seed(rows)
    q = (torch.randn((m, hq, dim), generator=g, device=DEV) * size).bfloat16()
    got = c8.attention(q, cache, table, i32(lens), cu_q=i32(cu), max_q=new, window=window)
    c8.check_status(DEV)
    want, room = attention64(q, cache, table, lens, cu, window)
    assert bool(got.isfinite().all())
    assert bool(((got.double() - want).abs() <= room).all())


@pytest.mark.parametrize("new,rows", HEADS)
def test_zero_and_tiny_rows_among_others(c8, new, rows):
    """Zero query rows beside ordinary ones, zero keys in some pages and ordinary ones in others."""
    hk, dim = 2, 128
    hq = hk * rows // new
    lens, cu = [200, 131], bounds([new] * 2)
    cache = filled_cache(c8, 8, hk, dim, 17 + rows)
    table = make_table(lens, 4, 8, rows)
    for page in (int(table[0, 3]), int(table[1, 0]), int(table[1, 2])):
        cache.k.view(torch.uint8)[page] = 0
        cache.k_exp[page] = 63
    q = torch.randn((2 * new, hq, dim), generator=torch.Generator(device=DEV).manual_seed(rows), device=DEV).bfloat16()
    q[:, ::2] = 0
    q[:, 1::4] *= 2.0**-100
    got = c8.attention(q, cache, table, i32(lens), cu_q=i32(cu), max_q=new)
    c8.check_status(DEV)
    want, room = attention64(q, cache, table, lens, cu)
    assert bool(((got.double() - want).abs() <= room).all())


@pytest.mark.parametrize("new,rows", HEADS)
def test_zero_rows_through_append_and_attention(c8, new, rows):
    """A layer fed with zeros (warm-up, zeroed padding slots): q, k and v are zero, and so is the result."""
    hk, dim = 2, 64
    hq = hk * rows // new
    cache = c8.new_cache(3, hk, dim, DEV)
    cos_sin, table = c8.rotary_table(dim, 2 * PAGE, DEV), i32([[2, 0], [1, 1]])
    x = torch.zeros((2 * new, (hq + 2 * hk) * dim), device=DEV, dtype=torch.bfloat16)
    lens, cu = i32([64 + new, new]), i32([0, new, 2 * new])
    q = c8.rope_append(x, cache, cos_sin, table, lens, q_heads=hq, cu_q=cu, max_q=new)
    out = c8.attention(q, cache, table, lens, cu_q=cu, max_q=new)
    c8.check_status(DEV)
    assert bool((out == 0).all())
