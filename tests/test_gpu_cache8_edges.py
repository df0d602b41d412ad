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


@pytest.mark.parametrize("new,rows", [(1, 8), (1, 16), (3, 24)])
@pytest.mark.parametrize("last", [False, True])
def test_many_small_weights_add_up(c8, new, rows, last):
    """One token that takes most, 400,000 others with 2^-25.5 of its weight each: together 0.8 % of the result. As many sequences
    as there are workers, so that each walks a whole sequence alone. Tolerance: the result's rounding (2^-8); each weight's
    rounding to FP16, at most half its smallest step, 2^-39 of the largest weight (2^-32 with 128-row tiles); FP32 sums of a
    term per page after one another, and 100 steps for what happens inside a page and the exponential."""
    n, dim, hq = 400000, 64, rows // new
    pages, batch = n // PAGE, torch.cuda.get_device_properties(DEV).multi_processor_count * (8 if rows <= 16 else 1)
    cache = c8.new_cache(2, 1, dim, DEV)   # all pages are page 1 but the one that holds the loud token
    one = 0x38   # 1.0
    cache.k.view(torch.uint8)[0, 0, 5, 0] = one
    cache.v.view(torch.uint8).fill_(one)
    cache.v.view(torch.uint8)[0, 0, dim // 2 :, 5] = 0
    q = torch.zeros((batch * new, hq, dim), device=DEV, dtype=torch.bfloat16)
    q[:, :, 0] = 1.0
    table = torch.ones((batch, pages), dtype=torch.int32, device=DEV)
    table[:, pages - 2 if last else 0] = 0
    lens, cu = torch.full((batch,), n, dtype=torch.int32, device=DEV), torch.arange(batch + 1, dtype=torch.int32, device=DEV) * new
    got = c8.attention(q, cache, table, lens, cu_q=cu, max_q=new, scale=25.5 * math.log(2.0)).double().view(batch, new, hq, dim)
    c8.check_status(DEV)
    weights = n * (2.0**-32 if rows > 16 else 2.0**-39) + (pages + 100) * 2.0**-24
    for j in range(new):
        rest = (n - new + j) * 2.0**-25.5
        for part, want in ((got[:, j, :, : dim // 2], 1.0), (got[:, j, :, dim // 2 :], rest / (1.0 + rest))):
            assert float((part - want).abs().max()) <= 2.0**-8 * want + weights, (j, want, float(part.min()), float(part.max()))


@pytest.mark.parametrize("new,rows", HEADS)
def test_scores_far_beyond_the_others(c8, new, rows):
    """Scores of 2^20 to 2^24, where a maximum's own rounding is worth powers of two, in rows beside zero rows: one token has
    all of a loud row's weight (the next is 2^19 and more below), a zero row is the mean of what it sees."""
    hk, dim, n = 2, 64, 150
    hq = hk * rows // new
    cache = filled_cache(c8, 3, hk, dim, 41)
    cache.k.view(torch.uint8).zero_()
    cache.k_exp.fill_(127)
    table = i32([[2, 0, 1]])
    for p, code in ((3, 0x34), (70, 0x38), (140, 0x36)):   # 0.75, 1, 0.875
        cache.k.view(torch.uint8)[int(table[0, p // PAGE]), :, p % PAGE, 0] = code
    q = torch.zeros((new, hq, dim), device=DEV, dtype=torch.bfloat16)
    q[:, 1::2, 0] = torch.exp2(torch.arange(hq // 2, device=DEV) % 4 + 12.0).bfloat16()
    got = c8.attention(q, cache, table, i32([n]), cu_q=i32([0, new]), max_q=new, scale=1023.0)
    c8.check_status(DEV)
    want, room = attention64(q, cache, table, [n], [0, new], scale=1023.0)
    top = values64_v(cache, table, 70).repeat_interleave(hq // hk, 0)[1::2]
    assert torch.equal(want.view(new, hq, dim)[:, 1::2], top.expand(new, -1, -1))
    assert bool(((got.double() - want).view(new, hq, dim)[:, 1::2].abs() <= 2.0**-8 * top.abs()).all())
    assert bool(((got.double() - want).abs() <= room).view(new, hq, dim)[:, ::2].all())


def values64_v(cache, table, p):
    page = int(table[0, p // PAGE])
    return cache.v[page, :, :, p % PAGE].double() * torch.exp2(cache.v_exp[page].double() - 127.0)[:, None]


def test_attention_half_in_8_bits_needs_no_bf16_weights(c8):
    """The BF16 weights may go once their 8-bit forms are made; without a form the call says so."""
    from llm_inference_engine_b200 import muse_bf16_proj as proj

    hq, hk, d, k = 4, 2, 64, 256
    g = torch.Generator(device=DEV).manual_seed(3)
    weights = {"qkv_gate": (0.05 * torch.randn(((2 * hq + 2 * hk) * d, k), generator=g, device=DEV)).bfloat16(),
               "o": (0.05 * torch.randn((k, hq * d), generator=g, device=DEV)).bfloat16()}
    state = proj.prepare(weights, warmup=False)
    cos_sin, table, lens = c8.rotary_table(64, PAGE, DEV), i32([[1], [0]]), i32([1, 1])
    x = torch.randn((2, k), generator=g, device=DEV).bfloat16()
    step = lambda: c8.attention_half({"x": x}, state, c8.new_cache(2, hk, d, DEV), cos_sin, table, lens, q_heads=hq, eight_bit=True)
    with pytest.raises(KeyError, match="prepare_fp8"):
        step()
    proj.prepare_fp8(state)
    before = step()
    del state["qkv_gate"], state["o"]
    assert torch.equal(step(), before)
    state["_fp8"]["o"] = tuple(t[:, :128] for t in state["_fp8"]["o"])
    with pytest.raises(ValueError, match="do not fit"):
        step()
    c8.check_status(DEV)


@pytest.mark.parametrize("most", [2**31 - 1, 1 << 20, 4096])
def test_max_q_may_be_any_bound(c8, most):
    """max_q is a bound: one far above what the batch holds gives what the batch's own row count gives."""
    hk, dim, hq = 2, 64, 8
    lens, new = [150, 64, 70], [3, 1, 0]
    cache = filled_cache(c8, 8, hk, dim, 77)
    table = make_table(lens, 3, 8, 1)
    x = torch.randn((4, (hq + 2 * hk) * dim), generator=torch.Generator(device=DEV).manual_seed(9), device=DEV).bfloat16()
    cu, cos_sin = i32(bounds(new)), c8.rotary_table(dim, 3 * PAGE, DEV)
    got = []
    for bound in (most, 4):
        held = type(cache)(*[t.clone() for t in cache])
        q = c8.rope_append(x, held, cos_sin, table, i32(lens), q_heads=hq, cu_q=cu, max_q=bound)
        got.append((c8.attention(q, held, table, i32(lens), cu_q=cu, max_q=bound), c8.attention(q, held, table, i32(lens), cu_q=cu, max_q=bound, out=torch.empty_like(q).flatten(1))))
    c8.check_status(DEV)
    assert all(torch.equal(t, got[1][0]) for pair in got for t in pair)
    want, room = attention64(q, held, table, lens, bounds(new))
    assert bool(((got[0][0].double() - want).abs() <= room).all())
