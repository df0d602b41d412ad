"""How the attention over the paged cache is dealt to workers (csrc/attn_sched.cuh), replayed on the host: every page
that a sequence's rows see is read exactly once per row tile and KV head, and the kernel that adds up partial sums finds
exactly the slots that were written, in page order. No GPU."""

from __future__ import annotations

import ctypes as C

import pytest

PAGE, WARPS = 64, 8


def plan(lens, cu, m, width, max_q, hq, hk, window, sms):
    from llm_inference_engine_b200 import _capi

    lib = _capi.load()
    ints = lambda v: (C.c_int * len(v))(*v) if v is not None else None
    lens_c, cu_c = ints(lens), ints(cu)
    args = (lens_c, cu_c, m, len(lens), width, max_q, hq, hk, window, sms)
    n = lib.muse_cache_attention_plan(*args, (C.c_int * 6)(), 0)
    assert n >= 0
    buf = (C.c_int * max(6 * n, 6))()
    assert lib.muse_cache_attention_plan(*args, buf, n) == n
    segs = [tuple(buf[6 * i : 6 * i + 6]) for i in range(n)]

    def join(entry, head):
        out = (C.c_int * 8192)()
        k = lib.muse_cache_attention_join(*args, entry, head, out, 8192)
        assert 0 <= k <= 8192
        return list(out[:k])

    return segs, join


def seen_pages(length, n, pos_lo, pos_hi, window):
    if pos_hi < 0:
        return [0]          # nothing is seen: one page that is masked whole
    lo = max(0, pos_lo - window + 1) if window else 0
    return list(range(lo // PAGE, pos_hi // PAGE + 1))


CASES = [
    # lens, new tokens (None: one each), width, hq, hk, window, sms
    ([300], None, 5, 32, 8, 0, 148),
    ([1], None, 1, 1, 1, 0, 148),
    ([0], None, 1, 4, 4, 0, 148),
    ([64, 65, 63, 0, 1], None, 2, 8, 4, 0, 3),
    ([100000, 100000], None, 1563, 32, 4, 0, 148),
    ([4000 - 37 * i for i in range(64)], None, 63, 32, 16, 0, 148),
    ([3001, 900, 1, 2, 64], [4, 0, 1, 2, 3], 47, 16, 4, 1000, 148),
    ([3001, 900, 4, 2000], [4, 3, 4, 0], 47, 16, 4, 1, 7),
    ([4096, 4096], [512, 512], 64, 32, 8, 0, 148),
    ([700, 50, 1300], [129, 50, 1], 21, 8, 1, 200, 5),
    ([3, 0], [5, 2], 1, 8, 8, 0, 4),          # more new tokens than tokens: padding rows
    ([64 * 1184 * 3], None, 1184 * 3, 4, 1, 0, 148),
    ([64 * 500, 64 * 37, 64 * 900 + 1], None, 1000, 16, 1, 0, 9),
    ([64 * 700 + i for i in range(5)], None, 1000, 8, 2, 0, 16),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{c[0][0]}_q{0 if c[1] is None else max(c[1])}_h{c[3]}-{c[4]}_w{c[5]}_s{c[6]}")
def test_every_page_is_read_once_and_joined_in_order(case):
    lens, new, width, hq, hk, window, sms = case
    cu = None if new is None else [sum(new[:i]) for i in range(len(new) + 1)]
    n = [1] * len(lens) if new is None else new
    m, max_q, group = sum(n), max(n), hq // hk
    segs, join = plan(lens, cu, m, width, max_q, hq, hk, window, sms)
    rows = max_q * group
    tile = 8 if rows <= 8 else 16 if rows <= 16 else 128
    tiles = -(-max_q * group // tile)
    units = {}
    for worker, entry, head, first, count, slot in segs:
        units.setdefault((entry, head), []).append((first, count, worker, slot))
    # a slot holds one segment, or the segments of a CTA's eight warps inside one unit, which are added up on chip
    slots = {}
    for i, s in enumerate(segs):
        if s[5] >= 0:
            slots.setdefault(s[5], []).append(i)
    for slot, where in slots.items():
        if len(where) > 1:
            same = [segs[i] for i in where]
            assert where == list(range(where[0], where[0] + WARPS)) and len({s[1:3] for s in same}) == 1
            assert [s[0] for s in same] == list(range(slot // 2, slot // 2 + WARPS)) and slot // 2 % WARPS == 0
    workers = sms if tile == 128 else sms * WARPS
    assert all(0 <= s[0] < workers for s in segs) and all(s < 2 * workers for s in slots)
    want = {}
    for b, (length, k) in enumerate(zip(lens, n)):
        for rt in range(tiles):
            r0, r1 = rt * tile, min((rt + 1) * tile, k * group)
            if r0 < r1:
                pos = length - k
                for h in range(hk):
                    want[b * tiles + rt, h] = seen_pages(length, k, pos + r0 // group, pos + (r1 - 1) // group, window)
    assert set(units) == set(want)
    share = [0] * workers
    for key, pages in want.items():
        parts = units[key]
        got = [p for first, count, _, _ in parts for p in range(first, first + count)]
        assert got == pages, (key, got, pages)
        if len(parts) == 1:
            assert parts[0][3] == -1 and join(*key) == []
        else:
            in_order = [p[3] for i, p in enumerate(parts) if i == 0 or parts[i - 1][3] != p[3]]
            assert in_order == join(*key) and all(s >= 0 for s in in_order)
        for _, count, w, _ in parts:
            share[w] += count
    # equal shares of items, a unit's pages and its two head items: no worker has more pages than its share of items
    items = sum(len(pages) + 2 for pages in want.values())
    assert all(share[w] <= -(-items // workers) for w in range(workers))
    assert sum(share) == sum(len(pages) for pages in want.values())


def test_bad_lengths_and_bounds_stay_inside():
    """Lengths beyond the table, falling or outlying bounds: whatever the tensors hold, pages stay inside the table and
    rows inside the batch."""
    for lens, cu in (([10 ** 6, -5], [0, 1, 2]), ([200, 100], [0, 5, 3]), ([200, 100], [-7, 1, 900]), ([200, 100], [2, 2, 2])):
        segs, _ = plan(lens, cu, 2, 4, 1, 8, 2, 0, 4)
        assert all(0 <= first and first + count <= 4 for _, _, _, first, count, _ in segs)
    from llm_inference_engine_b200 import _capi

    lib = _capi.load()
    one = (C.c_int * 2)(1, 1)
    buf = (C.c_int * 6)()
    for bad in (dict(hq=3, hk=2), dict(hk=0), dict(max_q=0), dict(width=0), dict(window=-1), dict(m=0), dict(sms=0)):
        a = dict(dict(m=1, batch=1, width=1, max_q=1, hq=2, hk=2, window=0, sms=4), **bad)
        assert lib.muse_cache_attention_plan(one, None, *[a[x] for x in ("m", "batch", "width", "max_q", "hq", "hk", "window", "sms")], buf, 1) < 0
