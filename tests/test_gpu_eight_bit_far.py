"""The 8-bit operators where addresses pass 32 bits: the last pages of a pool of 5 GB per tensor, and the last rows of a
result of 2.4 G values. The same call in a small place gives the same bits."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("new", [1, 5, 40])   # 2, 10 and 80 rows per KV head: tiles of 8, 16 and 128
def test_last_pages_of_a_large_pool(new):
    from llm_inference_engine_b200 import cache8

    if torch.cuda.mem_get_info(DEV)[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    heads, dim, hq, pages = 8, 128, 16, 80000
    assert (pages - 4) * heads * 64 * dim > 2**32
    far, near = cache8.new_cache(pages, heads, dim, DEV), cache8.new_cache(4, heads, dim, DEV)
    cos_sin = cache8.rotary_table(dim, 256, DEV)
    order = [2, 0, 3, 1]
    tables = [i32([[pages - 4 + p for p in order]]), i32([order])]
    g = torch.Generator(device=DEV).manual_seed(new)
    length, outs = 0, []
    for n in (150, new):
        length += n
        rows = torch.randn((n, (hq + 2 * heads) * dim), generator=g, device=DEV).bfloat16()
        outs = []
        for cache, table in zip((far, near), tables):
            batch = dict(cu_q=i32([0, n]), max_q=n)
            q = cache8.rope_append(rows, cache, cos_sin, table, i32([length]), q_heads=hq, **batch)
            outs.append(cache8.attention(q, cache, table, i32([length]), **batch))
        assert torch.equal(*outs) and bool(outs[0].isfinite().all()) and bool((outs[0] != 0).any())
    for a, b in zip(far, near):
        assert torch.equal(a[-4:].view(torch.uint8), b.view(torch.uint8))
        assert not bool((a[: pages % 65536].view(torch.uint8) != a[0].view(torch.uint8)).any())   # where a wrapped offset would land
    cache8.check_status(DEV)


def test_last_rows_of_a_large_result():
    from llm_inference_engine_b200 import fp8

    if torch.cuda.mem_get_info(DEV)[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    m, n, k = 200000, 12288, 144
    assert (m - 300) * n > 2**31
    g = torch.Generator(device=DEV).manual_seed(1)
    w8, we = fp8.quantize_weight(torch.randn((n, k), generator=g, device=DEV) * 0.02)
    x = torch.randn((m, k), generator=g, device=DEV).bfloat16()
    out = fp8.linear(x, w8, we)
    for at in (0, 2**31 // n - 100, m - 200):
        xv = fp8.quantize(x[at : at + 200])
        values = xv[0].double() * torch.exp2(xv[1].double() - 127).repeat_interleave(128, 1)[:, :k]
        want, mag = values @ fp8.dequantize_weight(w8, we).double().T, values.abs() @ fp8.dequantize_weight(w8, we).double().T.abs()
        # BF16's rounding, and 5 MMA steps of 32 columns, each cutting at 2^-23 of the sum of magnitudes
        assert bool(((out[at : at + 200].double() - want).abs() <= want.abs() * 2.0**-8 + mag * 6 * 2.0**-23).all())
