"""The rotary append to the 8-bit cache and the attention over it (cache8) against their definitions in 64 bits.

Tolerances. A rounding to type t is off by finfo(t).eps / 2 relative (BF16 2^-8, e4m3 2^-4, FP32 2^-24).
  rotation   FP32: each of two products and the sum rounded, and the table: 4 x 2^-24 of (|a| + |b|) amplitude; then BF16
             or e4m3 (half a code step: 2^-4 relative, 2^-10 of the scale below its normal range).
  attention  the result's BF16 rounding; P rounded to FP16 (2^-11 relative; 2^-25 of the largest below 2^-14 of it); scores
             from at most D / 16 + 4 MMA steps, each cutting at 2^-23 of the sum of magnitudes, in FP32 afterwards
             (2^-22 of the exponent's argument, the exponential's own 2^-21); sums of n tokens, n 2^-24. All but the
             first are relative to sum_p P |v| / sum_p P, which the reference computes beside the result.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
PAGE = 64


@pytest.fixture(scope="module")
def c8():
    from llm_inference_engine_b200 import cache8

    return cache8


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def values64(codes, byte):
    return codes.double() * torch.exp2(byte.double() - 127.0)[..., None, None]


def filled_cache(c8, pages, heads, dim, seed, spread=0.7):
    """A pool in use: quantised random values, heads of different magnitude."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = c8.new_cache(pages, heads, dim, DEV)
    for codes, byte in ((c.k, c.k_exp), (c.v, c.v_exp)):
        x = torch.randn(codes.shape, generator=g, device=DEV) * torch.exp(spread * torch.randn((pages, heads, 1, 1), generator=g, device=DEV))
        e = torch.ceil(torch.log2(x.abs().amax((2, 3)) / 448.0))
        codes.copy_((x / torch.exp2(e)[..., None, None]).clamp(-448, 448).to(torch.float8_e4m3fn))
        byte.copy_((e + 127).to(torch.uint8))
    return c


def clone(c):
    return type(c)(*[t.clone() for t in c])


def make_table(lens, width, pages, seed, capacity_rows=None):
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), width), 2 ** 30, dtype=torch.int32)      # unused places name no page
    for b, n in enumerate(lens):
        for i in range(-(-max(n, 0) // PAGE)):
            table[b, i] = order.pop()
    return table.to(DEV)


def bounds(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return cu


# ---------------------------------------------------------------- append

def rotate64(x, pos, rot, interleaved, base, scaling, factor, trained):
    """x [m, heads, dim] turned in 64 bits, from the formulas."""
    out = x.double().clone()
    amplitude = 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0
    for i in range(rot // 2):
        inv = base ** (-2.0 * i / rot)
        if scaling == "linear":
            inv /= factor
        elif scaling == "ntk":
            inv = (base * factor ** (rot / max(rot - 2, 1))) ** (-2.0 * i / rot)
        elif scaling == "yarn":
            keep = min(max((trained * inv / (2 * math.pi) - 1.0) / 31.0, 0.0), 1.0)
            inv *= keep + (1 - keep) / factor
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        c, s = amplitude * torch.cos(pos.double() * inv), amplitude * torch.sin(pos.double() * inv)
        xa, xb = x[..., a].double(), x[..., b].double()
        out[..., a] = xa * c[:, None] - xb * s[:, None]
        out[..., b] = xb * c[:, None] + xa * s[:, None]
    return out


def recode64(codes, ratio_log2):
    """e4m3 values times 2^ratio rounded to e4m3, in 64 bits."""
    y = codes.double() * 2.0 ** ratio_log2
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(y / step) * step


def check_append(c8, lens, new, hq, hk, dim, rot, interleaved=False, scaling="none", factor=4.0, trained=64, seed=0, width=None, with_cu=True, tweak=None,
                 view=True):
    m, cu = sum(new), bounds(new)
    width = width or max(1, max(-(-n // PAGE) for n in lens))
    pages = sum(-(-max(n, 0) // PAGE) for n in lens) + 3
    cache = filled_cache(c8, pages, hk, dim, seed)
    table = make_table(lens, width, pages, seed)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    cols = (hq + 2 * hk) * dim
    x = (torch.randn((m, cols), generator=g, device=DEV) * torch.exp(torch.randn((m, 1), generator=g, device=DEV))).bfloat16()
    if tweak:
        tweak(x)
    rows = torch.randn((m, cols + hq * dim), generator=g, device=DEV).bfloat16() if view else x
    if view:
        rows[:, :cols] = x
    before = clone(cache)
    cos_sin = c8.rotary_table(rot, width * PAGE, DEV, scaling=scaling, factor=factor, trained_positions=trained)
    q, kv, vv = c8.rope_append(rows, cache, cos_sin, table, i32(lens), q_heads=hq, cu_q=i32(cu) if with_cu else None, max_q=max(new), interleaved=interleaved,
                               values=True)
    torch.cuda.synchronize(DEV)
    c8.check_status(DEV)
    pos = torch.cat([torch.arange(n - k, n) for n, k in zip(lens, new)]).to(DEV)
    heads = x.double().view(m, -1, dim)
    turned = rotate64(heads[:, : hq + hk], pos, rot, interleaved, 10000.0, scaling, factor, trained)
    amp = 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0
    mags = heads[:, : hq + hk].abs()
    partner = mags.clone()
    if interleaved:
        partner[..., 0:rot:2], partner[..., 1:rot:2] = mags[..., 1:rot:2], mags[..., 0:rot:2]
    else:
        partner[..., : rot // 2], partner[..., rot // 2 : rot] = mags[..., rot // 2 : rot], mags[..., : rot // 2]
    slack = 4 * 2.0 ** -24 * amp * (mags + partner)
    inside = (pos >= 0)[:, None, None]
    want_q = torch.where(inside, turned[:, :hq], torch.zeros_like(turned[:, :hq]))
    fine = want_q.isfinite()
    assert torch.equal(q.isfinite(), fine)
    off = (q.double() - want_q).abs()
    assert bool((off[fine] <= (2.0 ** -8 * want_q.abs() + 2 * slack[:, :hq])[fine]).all())
    # the cache, page by page
    expect_same = [t.clone() for t in before]
    for b, (n, k) in enumerate(zip(lens, new)):
        start = max(n - k, 0)
        for pg in range(start // PAGE, -(-n // PAGE) if n > 0 else 0):
            page = int(table[b, pg])
            s0, s1 = max(start, pg * PAGE) - pg * PAGE, min(n, (pg + 1) * PAGE) - pg * PAGE
            if s0 >= s1:
                continue
            r0 = cu[b] + pg * PAGE + s0 - (n - k)
            for h in range(hk):
                for name, y, sl in (("k", turned[r0 : r0 + s1 - s0, hq + h], slack[r0 : r0 + s1 - s0, hq + h]),
                                    ("v", heads[r0 : r0 + s1 - s0, hq + hk + h], torch.zeros((s1 - s0, dim), device=DEV, dtype=torch.float64))):
                    codes, byte = getattr(cache, name), getattr(cache, name + "_exp")
                    old, oldb = getattr(before, name), getattr(before, name + "_exp")
                    held = codes[page, h].double() if name == "k" else codes[page, h].double().T      # [token, dim]
                    was = old[page, h].double() if name == "k" else old[page, h].double().T
                    e = int(byte[page, h]) - 127
                    ok = y.isfinite()
                    a = float(y[ok].abs().max()) if bool(ok.any()) else 0.0
                    room = float(sl[ok].max()) if bool(ok.any()) else 0.0
                    floor = int(oldb[page, h]) - 127 if s0 else -64
                    assert e >= floor and 448.0 * 2.0 ** e >= a - room, (name, page, h, e, a)
                    assert e == floor or 448.0 * 2.0 ** (e - 1) < a + room, (name, page, h, e, a)
                    got = held[s0:s1] * 2.0 ** e
                    assert torch.equal(got.isfinite(), ok)
                    step = torch.maximum(2.0 ** -4 * y.abs(), torch.full_like(y, 2.0 ** (e - 10)))
                    assert bool(((got - y).abs()[ok] <= (step + 2 * sl)[ok]).all()), (name, page, h)
                    val = (kv if name == "k" else vv)[r0 : r0 + s1 - s0, h].double()
                    assert torch.equal(val[ok], got[ok]) and torch.equal(val.isfinite(), ok)
                    if s0:
                        moved = recode64(was[:s0], (int(oldb[page, h]) - 127) - e)
                        assert torch.equal(held[:s0], moved), (name, page, h)
                    assert torch.equal(held[s1:], was[s1:]), "tokens behind the sequence stay as they were"
                    i = ("k", "v").index(name)
                    expect_same[i][page, h] = codes[page, h]
                    expect_same[2 + i][page, h] = byte[page, h]
    for got, want in zip(cache, expect_same):
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8)), "a page that belongs to nobody's new tokens has changed"
    pad = pos < 0
    assert bool((kv[pad] == 0).all()) and bool((vv[pad] == 0).all())
    return cache, before


APPENDS = [
    dict(lens=[1], new=[1], hq=1, hk=1, dim=64, rot=64),
    dict(lens=[1, 64, 65, 128, 500], new=[1] * 5, hq=8, hk=2, dim=128, rot=128, with_cu=False),
    dict(lens=[70, 64, 3, 200, 129], new=[5, 0, 3, 1, 4], hq=6, hk=3, dim=64, rot=32, interleaved=True, scaling="linear"),
    dict(lens=[63 + 16, 64 + 7], new=[16, 16], hq=4, hk=4, dim=128, rot=16, scaling="ntk"),
    dict(lens=[17, 80, 300], new=[17, 17, 17], hq=8, hk=1, dim=128, rot=64, interleaved=True, scaling="yarn"),
    dict(lens=[64, 192, 321], new=[64, 128, 257], hq=2, hk=2, dim=128, rot=128, scaling="yarn", view=False),
    dict(lens=[640], new=[600], hq=4, hk=2, dim=64, rot=48),
    dict(lens=[2, 0, 1], new=[5, 2, 1], hq=4, hk=2, dim=64, rot=64, width=2),                  # padding rows
    dict(lens=[90000], new=[3], hq=2, hk=1, dim=128, rot=128, scaling="linear"),               # far positions
]


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"q{max(c['new'])}_len{max(c['lens'])}_h{c['hq']}-{c['hk']}_d{c['dim']}r{c['rot']}")
def test_append_matches_64_bits(c8, case):
    check_append(c8, seed=sum(case["lens"]), **case)


def test_append_what_is_not_finite_zero_tiny_and_huge(c8):
    def tweak(x):
        x[0, 4 * 64 + 3] = float("nan")        # k of head 0
        x[1, 6 * 64 + 9] = float("inf")        # v of head 0
        x[2] = 0
        x[3] = 2.0 ** -90
        x[4, 4 * 64 :] *= 2.0 ** 100
    check_append(c8, [70, 71, 64, 65, 130], [1] * 5, 4, 2, 64, 64, seed=9, tweak=tweak)


def test_a_page_filled_token_by_token_keeps_its_largest_scale(c8):
    """64 appends of one token with growing and falling magnitudes: every code is the value rounded once to the scale of
    its own time and then recoded; the exponent is the running largest."""
    cache = c8.new_cache(2, 1, 64, DEV)
    table, cos_sin = i32([[1]]), c8.rotary_table(64, 64, DEV)
    top = -64
    for p in range(64):
        x = (torch.randn((1, 3 * 64), device=DEV) * 2.0 ** ((p * 7) % 13)).bfloat16()
        before = clone(cache)
        c8.rope_append(x, cache, cos_sin, table, i32([p + 1]), q_heads=1)
        e = math.ceil(math.log2(float(x[0, 128:].float().abs().max()) / 448.0))
        top = max(top, e)
        assert int(cache.v_exp[1, 0]) - 127 == top
        assert torch.equal(cache.v[1, 0].double()[:, :p], recode64(before.v[1, 0].double()[:, :p], int(before.v_exp[1, 0]) - 127 - top))
        assert bool(((cache.v[1, 0, :, p].double() * 2.0 ** top - x[0, 128:].double()).abs() <= torch.maximum(2.0 ** -4 * x[0, 128:].double().abs(), torch.tensor(2.0 ** (top - 10)))).all())
    c8.check_status(DEV)
    # the same page again from its first token: the scale starts afresh
    x = (torch.randn((1, 3 * 64), device=DEV) * 2.0 ** -3).bfloat16()
    c8.rope_append(x, cache, cos_sin, table, i32([1]), q_heads=1)
    assert int(cache.v_exp[1, 0]) - 127 == math.ceil(math.log2(float(x[0, 128:].float().abs().max()) / 448.0))


# ---------------------------------------------------------------- attention

def attention64(q, cache, table, lens, cu, window=0, gate=None, scale=None):
    """(o, allowance) in 64 bits, from the definition: [m, hq * dim] each."""
    m, hq, d = q.shape
    hk = cache.k.shape[1]
    out, room = torch.zeros((m, hq, d), dtype=torch.float64, device=DEV), torch.zeros((m, hq, d), dtype=torch.float64, device=DEV)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    for b, n in enumerate(lens):
        if n <= 0 or cu[b] == cu[b + 1]:
            continue
        idx = table[b, : -(-n // PAGE)].long()
        pos = torch.arange(n - (cu[b + 1] - cu[b]), n, device=DEV)[:, None]
        j = torch.arange(n, device=DEV)[None, :]
        seen = (j <= pos) & ((j > pos - window) if window else (j >= 0))
        for h in range(hk):
            k = values64(cache.k[idx, h], cache.k_exp[idx, h]).reshape(-1, d)[:n]
            v = values64(cache.v[idx, h], cache.v_exp[idx, h]).transpose(1, 2).reshape(-1, d)[:n]
            for a in range(h * (hq // hk), (h + 1) * (hq // hk)):
                qa = q[cu[b] : cu[b + 1], a].double()
                s = torch.where(seen, scale * (qa @ k.T), torch.full((), -math.inf, dtype=torch.float64, device=DEV))
                none = ~seen.any(-1, keepdim=True)
                p = torch.exp(s - torch.where(none, torch.zeros_like(s[:, :1]), s.amax(-1, keepdim=True)))
                p = torch.where(seen, p, torch.zeros_like(p)) / torch.where(none, torch.ones_like(s[:, :1]), p.sum(-1, keepdim=True))
                # a token that a row does not see has no part in it, whatever it holds
                o = torch.zeros((p.shape[0], d), dtype=torch.float64, device=DEV)
                mag = torch.zeros_like(o)
                for r in range(p.shape[0]) if not bool(v.isfinite().all()) else []:
                    o[r], mag[r] = p[r, seen[r]] @ v[seen[r]], p[r, seen[r]] @ v[seen[r]].abs()
                if bool(v.isfinite().all()):
                    o, mag = p @ v, p @ v.abs()
                big = scale * (qa.abs() @ torch.nan_to_num(k).abs().T).masked_fill(~seen, 0).amax(-1, keepdim=True)
                rel = 2.0 ** -11 + 4 * (d / 16 + 4) * 2.0 ** -23 * big + 2.0 ** -20 + n * 2.0 ** -24
                out[cu[b] : cu[b + 1], a] = o
                room[cu[b] : cu[b + 1], a] = 2 * rel * mag + 2.0 ** -25 * v.nan_to_num().abs().amax() / p.clamp(min=1e-9).amax(-1, keepdim=True).clamp(min=2.0 ** -20)
    if gate is not None:
        s = torch.sigmoid(gate.double()).view(m, hq, d)
        out, room = out * s, room * s + 2.0 ** -20 * (out * s).abs()
    return out.flatten(1), (room + 2.0 ** -8 * out.abs()).flatten(1)


def check_attention(c8, lens, new, hq, hk, dim, window=0, gated=False, seed=0, with_cu=True, pages=None, spread=0.7, poison=True, scale=None, loud=1.0):
    m, cu = sum(new), bounds(new)
    need = sum(-(-max(n, 0) // PAGE) for n in lens)
    cache = filled_cache(c8, need + 2, hk, dim, seed, spread)
    width = max(1, max(-(-n // PAGE) for n in lens)) + 1
    table = make_table(lens, width, need + 2, seed)
    if poison:      # what lies behind a sequence's last token in its last page may be anything
        for b, n in enumerate(lens):
            if n > 0 and n % PAGE:
                last = int(table[b, n // PAGE])
                cache.k.view(torch.uint8)[last, :, n % PAGE :] = 0x7F
                cache.v.view(torch.uint8)[last, :, :, n % PAGE :] = 0xFF
    g = torch.Generator(device=DEV).manual_seed(seed + 5)
    q = (loud * torch.randn((m, hq, dim), generator=g, device=DEV)).bfloat16()
    wide = torch.randn((m, 3 * hq * dim), generator=g, device=DEV).bfloat16()
    gate = wide[:, hq * dim : 2 * hq * dim] if gated else None
    out = torch.full((m + 2, hq * dim), 5.0, device=DEV, dtype=torch.bfloat16)
    got = c8.attention(q, cache, table, i32(lens), cu_q=i32(cu) if with_cu else None, max_q=max(new), window=window, gate=gate, out=out[1:-1], scale=scale)
    torch.cuda.synchronize(DEV)
    c8.check_status(DEV)
    want, room = attention64(q, cache, table, lens, cu, window, gate, scale)
    assert torch.equal(got.isfinite(), want.isfinite())
    off = (got.double() - want).abs() - room
    assert float(off.max()) <= 0, f"off by {float((got.double() - want).abs().max()):.3g}, {float(off.max()):.3g} more than allowed"
    assert bool((out[0] == 5).all()) and bool((out[-1] == 5).all())
    again = c8.attention(q, cache, table, i32(lens), cu_q=i32(cu) if with_cu else None, max_q=max(new), window=window, gate=gate, scale=scale)
    assert torch.equal(again, got), "two runs differ"


ATTENTIONS = [
    dict(lens=[1], new=[1], hq=1, hk=1, dim=128),
    dict(lens=[300], new=[1], hq=32, hk=8, dim=128, gated=True, with_cu=False),
    dict(lens=[64, 65, 63, 1, 128, 2000], new=[1] * 6, hq=16, hk=2, dim=128, with_cu=False),
    dict(lens=[64, 65, 63, 1, 128, 2000], new=[1] * 6, hq=8, hk=8, dim=64, gated=True, with_cu=False),
    dict(lens=[0, 5, 0], new=[1, 1, 1], hq=4, hk=2, dim=64, with_cu=False),                     # rows that see nothing
    dict(lens=[3000, 900, 4, 2000], new=[4, 3, 4, 0], hq=16, hk=4, dim=64, window=100),
    dict(lens=[3000, 900, 4, 2000], new=[4, 3, 4, 1], hq=8, hk=2, dim=128, window=1),
    dict(lens=[500, 2, 77], new=[3, 5, 7], hq=2, hk=1, dim=128, gated=True),                     # 14 rows; padding rows
    dict(lens=[40000], new=[1], hq=16, hk=1, dim=128),
    dict(lens=[20000, 3], new=[2, 1], hq=16, hk=2, dim=64, window=15000),
    dict(lens=[200, 64, 1000], new=[130, 64, 9], hq=8, hk=2, dim=128, gated=True),               # a CTA's 128-row tiles
    dict(lens=[200, 90, 1000, 30], new=[17, 0, 100, 40], hq=4, hk=4, dim=64, window=50),
    dict(lens=[700], new=[513], hq=4, hk=1, dim=64),
    dict(lens=[300, 20], new=[3, 3], hq=32, hk=1, dim=128),                                      # 96 rows of one head
    dict(lens=[7 * i + 1 for i in range(70)], new=[1] * 70, hq=4, hk=4, dim=64, with_cu=False),
    dict(lens=[13 * i % 300 for i in range(300)], new=[1] * 300, hq=8, hk=1, dim=128, with_cu=False),
]


@pytest.mark.parametrize("case", ATTENTIONS, ids=lambda c: f"b{len(c['lens'])}_len{max(c['lens'])}_q{max(c['new'])}_h{c['hq']}-{c['hk']}_d{c['dim']}_w{c.get('window', 0)}")
def test_attention_matches_64_bits(c8, case):
    check_attention(c8, seed=sum(case["lens"]), **case)


def test_attention_scales_and_magnitudes(c8):
    """Pages whose scales differ by e^(4 sigma), loud queries (one token takes nearly all), a scale of its own."""
    check_attention(c8, [700, 90], [1, 1], 8, 2, 128, seed=3, spread=3.0)
    check_attention(c8, [700, 90], [2, 1], 8, 2, 64, seed=4, spread=3.0, loud=8.0)
    check_attention(c8, [700, 90], [30, 1], 8, 2, 64, seed=5, loud=4.0, scale=0.3)
    check_attention(c8, [700], [1], 8, 2, 64, seed=6, scale=2.0 ** -20)


def test_nan_in_a_token_reaches_only_the_rows_that_see_it(c8):
    """A drafted token whose v (and another whose k) is NaN: the rows before it stay finite, in both tile forms."""
    for new, hq, hk in ((4, 4, 2), (40, 8, 2)):
        n, d = 150, 64
        cache = filled_cache(c8, 4, hk, d, 11)
        table = i32([[2, 0, 3]])
        p = n - new + 2
        cache.v.view(torch.uint8)[int(table[0, p // PAGE]), 0, 5, p % PAGE] = 0x7F
        cache.k.view(torch.uint8)[int(table[0, (p + 1) // PAGE]), 1, (p + 1) % PAGE, 7] = 0xFF
        q = torch.randn((new, hq, d), device=DEV).bfloat16()
        got = c8.attention(q, cache, table, i32([n]), cu_q=i32([0, new]), max_q=new)
        want, room = attention64(q, cache, table, [n], [0, new])
        assert torch.equal(got.isnan(), want.isnan()) and bool(want.isnan().any()) and not bool(want[:2].isnan().any())
        fine = ~want.isnan()
        assert bool(((got.double() - want).abs() <= room)[fine].all())


def test_shared_prefix_strided_and_misaligned_inputs(c8):
    """Two sequences that read the same pages; q as a slice of wider rows and misaligned; gate misaligned."""
    cache = filled_cache(c8, 6, 2, 64, 21)
    table = i32([[0, 1, 2, 3], [0, 1, 2, 4], [0, 1, 5, 5]])
    lens, cu = [200, 230, 130], [0, 1, 2, 3]
    rows = torch.randn((3, 8 * 64 * 2 + 8), device=DEV).bfloat16()
    q = rows[:, 8 : 8 + 512].unflatten(1, (8, 64))
    gate = rows[:, 515 : 515 + 512]
    got = c8.attention(q, cache, table, i32(lens), gate=gate)
    want, room = attention64(q, cache, table, lens, cu, gate=gate)
    assert bool(((got.double() - want).abs() <= room).all())
    odd = rows[:, 3 : 3 + 512].unflatten(1, (8, 64))
    assert torch.equal(c8.attention(odd, cache, table, i32(lens)), c8.attention(odd.contiguous(), cache, table, i32(lens)))


def test_bad_pages_and_lengths_are_reported_and_masked(c8):
    """An index outside the pool is neither read nor written, and the call says so; the other sequences are right."""
    cache = filled_cache(c8, 4, 2, 64, 31)
    before = clone(cache)
    table = i32([[0, 7], [1, 2]])
    q = torch.randn((2, 4, 64), device=DEV).bfloat16()
    got = c8.attention(q, cache, table, i32([100, 128]))
    with pytest.raises(Exception, match="page index outside"):
        c8.check_status(DEV)
    want, room = attention64(q, cache, i32([[0, 0], [1, 2]]), [64, 128], [0, 1, 2])      # the bad page counts as masked
    assert bool(((got.double() - want).abs() <= room).all())
    got = c8.attention(q, cache, i32([[0, 3], [1, 2]]), i32([129, 128]))
    with pytest.raises(Exception, match="lengths"):
        c8.check_status(DEV)
    want, room = attention64(q[1:], cache, i32([[1, 2]]), [128], [0, 1])
    assert bool(((got[1:].double() - want).abs() <= room).all())
    cos_sin = c8.rotary_table(64, 128, DEV)
    x = torch.randn((2, 8 * 64), device=DEV).bfloat16()
    qr, kv, vv = c8.rope_append(x, cache, cos_sin, i32([[0, -1], [1, 2]]), i32([100, 129]), q_heads=4, values=True)
    with pytest.raises(Exception, match="page index outside.*lengths"):
        c8.check_status(DEV)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, before))
    assert bool((kv == 0).all()) and bool((vv == 0).all()) and bool((qr[1] == 0).all())
    c8.check_status(DEV)


def test_rows_behind_the_last_sequence_stay(c8):
    cache = filled_cache(c8, 4, 2, 64, 41)
    q = torch.randn((6, 4, 64), device=DEV).bfloat16()
    out = torch.full((6, 256), 3.0, device=DEV, dtype=torch.bfloat16)
    c8.attention(q, cache, i32([[0], [1]]), i32([10, 20]), cu_q=i32([0, 1, 4]), max_q=4, out=out)
    c8.check_status(DEV)
    assert bool((out[4:] == 3).all()) and not bool((out[:4] == 3).any())


def test_replay_with_other_lengths_and_two_graphs_at_once(c8):
    """One step (append, attention) captured twice, each graph with buffers of its own over a pool of its own, replayed at
    once on two streams while lengths grow: the bits of eager steps."""
    hq, hk, d, b = 8, 2, 64, 5
    cos_sin = c8.rotary_table(64, 4 * PAGE, DEV)
    table = torch.arange(20, dtype=torch.int32, device=DEV).view(5, 4)
    steps = [(torch.randn((b, (2 * hq + 2 * hk) * d), device=DEV)).bfloat16() for _ in range(12)]
    first = [1, 60, 64, 120, 30]

    def step(rows, cache, lens):
        q = c8.rope_append(rows, cache, cos_sin, table, lens, q_heads=hq)
        return c8.attention(q, cache, table, lens, gate=rows[:, (hq + 2 * hk) * d :])

    eager_cache = filled_cache(c8, 20, hk, d, 51)
    start = clone(eager_cache)
    want = [step(rows, eager_cache, i32([n + i for n in first])).clone() for i, rows in enumerate(steps)]
    torch.cuda.synchronize(DEV)
    graphs = []
    for _ in range(2):
        cache, rows, lens = clone(start), steps[0].clone(), i32(first)
        side = torch.cuda.Stream(DEV)
        side.wait_stream(torch.cuda.current_stream(DEV))
        with torch.cuda.stream(side):
            step(rows, clone(start), lens)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step(rows, cache, lens)
        graphs.append((g, side, cache, rows, lens, out))
    for i, x in enumerate(steps):
        torch.cuda.synchronize(DEV)
        for g, side, cache, rows, lens, out in graphs:
            with torch.cuda.stream(side):
                rows.copy_(x)
                lens.copy_(i32([n + i for n in first]))
                g.replay()
        torch.cuda.synchronize(DEV)
        for g, side, cache, rows, lens, out in graphs:
            assert torch.equal(out, want[i]), i
    for g, side, cache, rows, lens, out in graphs:
        assert all(torch.equal(a.view(torch.uint8), e.view(torch.uint8)) for a, e in zip(cache, eager_cache))
    c8.check_status(DEV)


def test_refusals(c8):
    cache = filled_cache(c8, 4, 2, 64, 61)
    table, lens = i32([[0, 1], [2, 3]]), i32([5, 70])
    q = torch.randn((2, 4, 64), device=DEV).bfloat16()
    rows = torch.randn((2, 8 * 64), device=DEV).bfloat16()
    cs = c8.rotary_table(64, 128, DEV)
    bad_attention = [
        (TypeError, dict(q=q.float())), (TypeError, dict(q=q[0])), (ValueError, dict(q=torch.zeros((2, 4, 128), device=DEV, dtype=torch.bfloat16))),
        (ValueError, dict(q=q[:, :3])), (ValueError, dict(q=q[:1])), (TypeError, dict(page_table=table.long())), (ValueError, dict(seq_lens=lens[:1])),
        (TypeError, dict(seq_lens=lens.cpu())), (ValueError, dict(cu_q=i32([0, 1]))), (ValueError, dict(max_q=2)), (ValueError, dict(max_q=0, cu_q=i32([0, 1, 2]))),
        (ValueError, dict(window=-1)), (ValueError, dict(scale=0.0)), (ValueError, dict(scale=-1.0)), (TypeError, dict(gate=q.flatten(1).float())), (TypeError, dict(gate=q.flatten(1)[:, :8])),
        (ValueError, dict(out=torch.empty((256, 2), device=DEV, dtype=torch.bfloat16).T)),
        (ValueError, dict(cache=cache._replace(v=cache.v[:3]))), (TypeError, dict(cache=cache._replace(k=cache.k.view(torch.uint8)))),
        (ValueError, dict(cache=cache._replace(k_exp=cache.k_exp[:3]))),
    ]
    for error, change in bad_attention:
        a = dict(dict(q=q, cache=cache, page_table=table, seq_lens=lens), **change)
        with pytest.raises(error):
            c8.attention(a.pop("q"), a.pop("cache"), a.pop("page_table"), a.pop("seq_lens"), **a)
    bad_append = [
        (TypeError, dict(qkv=rows.float())), (ValueError, dict(qkv=rows[:, :500])), (ValueError, dict(qkv=rows[:1])), (ValueError, dict(cos_sin=cs[:127])),
        (TypeError, dict(cos_sin=cs.double())), (ValueError, dict(cos_sin=c8.rotary_table(8, 128, DEV))), (ValueError, dict(cos_sin=c8.rotary_table(80, 128, DEV))),
        (ValueError, dict(q_heads=5)), (ValueError, dict(q_heads=1)), (ValueError, dict(cos_sin=cs.cpu())),
    ]
    for error, change in bad_append:
        a = dict(dict(qkv=rows, cos_sin=cs, q_heads=4), **change)
        with pytest.raises(error):
            c8.rope_append(a["qkv"], cache, a["cos_sin"], table, lens, q_heads=a["q_heads"])
    for kw in (dict(scaling="yarn", factor=2.0), dict(scaling="other"), dict(factor=0.5)):
        with pytest.raises(ValueError):
            c8.rotary_table(64, 10, DEV, **kw)
    with pytest.raises(ValueError):
        c8.new_cache(4, 2, 96, DEV)
    cpu = c8.Cache8(*[t.cpu() for t in cache])
    with pytest.raises(RuntimeError, match="CUDA device only"):
        c8.attention(q.cpu(), cpu, table.cpu(), lens.cpu())
    c8.check_status(DEV)


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("eight_bit", [False, True])
def test_attention_half_of_a_layer_over_a_prompt_and_steps(c8, eight_bit):
    """A prompt of ragged sequences, then single tokens, then drafts, through attention_half: against the same stages in 64
    bits, each fed with what the stage before it gave (the stages' own tolerances)."""
    from llm_inference_engine_b200 import fp8, muse_bf16_proj as proj

    hq, hk, d, k = 8, 2, 64, 512
    g = torch.Generator(device=DEV).manual_seed(71)
    weights = {"qkv_gate": (0.05 * torch.randn(((2 * hq + 2 * hk) * d, k), generator=g, device=DEV)).bfloat16(),
               "o": (0.05 * torch.randn((k, hq * d), generator=g, device=DEV)).bfloat16()}
    state = proj.prepare(weights, warmup=False)
    if eight_bit:
        proj.prepare_fp8(state)
    cache = c8.new_cache(16, hk, d, DEV)
    table = torch.arange(15, dtype=torch.int32, device=DEV).view(3, 5).flip(1).contiguous()
    cos_sin = c8.rotary_table(64, 5 * PAGE, DEV)
    lens = [0, 0, 0]
    for new in ([100, 64, 3], [1, 1, 1], [1, 1, 1], [4, 0, 2], [1, 1, 1]):
        lens = [a + b for a, b in zip(lens, new)]
        m, cu = sum(new), bounds(new)
        x = torch.randn((m, k), generator=g, device=DEV).bfloat16()
        one = all(n == 1 for n in new)
        got = c8.attention_half({"x": x}, state, cache, cos_sin, table, i32(lens), q_heads=hq, cu_q=None if one else i32(cu), max_q=max(new), eight_bit=eight_bit)
        project = proj.kernel_fn_fp8 if eight_bit else proj.kernel_fn
        rows = project({"x": x, "config": {"layer": "qkv_gate", "m": m, "n": weights["qkv_gate"].shape[0], "k": k}}, state)
        qkv = (hq + 2 * hk) * d
        pos = torch.cat([torch.arange(n - c, n) for n, c in zip(lens, new)]).to(DEV)
        q = rotate64(rows[:, : hq * d].view(m, hq, d), pos, 64, False, 10000.0, "none", 1.0, None).bfloat16()
        a, room = attention64(q, cache, table, lens, cu, gate=rows[:, qkv:])
        o = (fp8.dequantize_weight(*state["_fp8"]["o"]) if eight_bit else weights["o"]).double()
        want = a @ o.T
        # what the stages before allow, through |o|; in 8 bits also the rounding of a to codes (2^-4 of a value, 2^-10 of
        # its block's scale, which is at most 2 * amax / 448)
        if eight_bit:
            room = room * 2 + 2.0 ** -4 * a.abs() + 2.0 ** -10 * 2 * a.abs().amax() / 448.0 * 2
        # q was rounded to BF16 from FP32 and from 64 bits: one BF16 step apart at most, 2^-8 of a score's magnitude
        big = 2.0 ** -8 * 2 * a.abs().amax()
        allow = (room + big) @ o.abs().T + 2.0 ** -8 * want.abs() + hq * d * 2.0 ** -23 * (a.abs() @ o.abs().T)
        assert bool(((got.double() - want).abs() <= allow).all())
    c8.check_status(DEV)
    proj.check_status(state)


def test_first_call_of_a_device_inside_a_capture_is_refused(c8):
    """The status word is made by the first call and has to outlive every graph."""
    from llm_inference_engine_b200 import _capi

    cache = filled_cache(c8, 2, 1, 64, 81)
    q = torch.randn((1, 1, 64), device=DEV).bfloat16()
    table, lens = i32([[0]]), i32([5])
    torch.cuda.synchronize(DEV)
    kept = _capi._STATUS.pop(DEV.index, None)
    _capi.bind().set_status(DEV.index, 0)
    try:
        g = torch.cuda.CUDAGraph()
        with pytest.raises(_capi.MuseError, match="outside stream capture"):
            with torch.cuda.graph(g):
                c8.attention(q, cache, table, lens)
    finally:
        if kept is not None:
            _capi._STATUS[DEV.index] = kept
            _capi.bind().set_status(DEV.index, kept.data_ptr())
    torch.cuda.synchronize(DEV)
    c8.attention(q, cache, table, lens)
    c8.check_status(DEV)


def test_ordinary_calls_take_the_short_way_and_give_the_same_bits(c8, monkeypatch):
    """What csrc/bind.cpp takes and what the Python code does with the same arguments: equal results, equal cache."""
    from llm_inference_engine_b200 import _capi, fp8

    class Never:
        linear = rope_append = attention = staticmethod(lambda *a: None)
        set_status = staticmethod(lambda *a: None)

    hq, hk, d = 8, 2, 64
    cos_sin = c8.rotary_table(64, 4 * PAGE, DEV)
    table = torch.arange(12, dtype=torch.int32, device=DEV).view(3, 4)
    x = torch.randn((3, 512), device=DEV).bfloat16()
    w8, we = fp8.quantize_weight(torch.randn(((2 * hq + 2 * hk) * d, 512), device=DEV))
    start = filled_cache(c8, 12, hk, d, 91)

    def run(cache):
        rows = fp8.linear(x, w8, we)
        many = fp8.linear(x.repeat(30, 1), w8, we)
        q, kv, vv = c8.rope_append(rows, cache, cos_sin, table, i32([3, 70, 128]), q_heads=hq, values=True)
        q2 = c8.rope_append(rows, cache, cos_sin, table, i32([3, 70, 0]), q_heads=hq, cu_q=i32([0, 2, 3, 3]), max_q=2, interleaved=True)
        a = c8.attention(q, cache, table, i32([3, 70, 128]), gate=rows[:, (hq + 2 * hk) * d :], window=50, scale=0.2)
        return [rows, many, q, kv, vv, q2, a, *[t.view(torch.uint8) for t in cache]]

    run(clone(start))
    b = _capi.bind()
    q = torch.randn((3, hq, d), device=DEV).bfloat16()
    assert b.attention(q, start, table, i32([3, 70, 128]), None, 1, None, 0, None) is not None
    assert b.linear(x, w8, we) is not None
    for args in ((q.float(), start, table, i32([3, 70, 128]), None, 1, None, 0, None), (q, start, table, i32([3, 70]), None, 1, None, 0, None),
                 (q, start, table, i32([3, 70, 128]), None, 2, None, 0, None), (q, start, table, i32([3, 70, 128]), None, 1, -1.0, 0, None),
                 (q, start, table, i32([3, 70, 128]), None, 1, None, -1, None), (q, list(start), table, i32([3, 70, 128]), None, 1, None, 0, None),
                 (None, start, table, i32([3, 70, 128]), None, 1, None, 0, None), (q, start)):
        assert b.attention(*args) is None, "not an ordinary call"
    short = run(clone(start))
    monkeypatch.setattr(_capi, "_BIND", Never)
    long_way = run(clone(start))
    assert all(torch.equal(u, w) for u, w in zip(short, long_way))
    c8.check_status(DEV)
