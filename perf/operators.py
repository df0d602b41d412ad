"""What the 8-bit operators of the decode layer's attention half are measured on: the block-scaled 8-bit
projection, the rotary step that appends keys and values to an 8-bit cache, and the attention that reads it.

Each case is one call as a serving program makes it. `run` computes it from elementary torch operations in
FP32, or, where `own` is true, through the framework's entry points on the same inputs.

Number formats, shared by all three operators: an 8-bit value is an e4m3 code times a power of two; the exponent
of a block whose largest finite magnitude is a is e = max(ceil(log2(a / 448)), -64), stored as the byte e + 127;
codes are rounded to nearest even, values that are not finite become NaN.
  projection   x and W: one exponent per token and 128 columns, and per 128 x 128 block of W
  cache        pages of 64 tokens; one exponent per page and head for K ([page, head, token, dim]) and one for V
               ([page, head, dim, token]); a page's exponent never falls while the page fills: when a new token
               raises it, the codes of the page's earlier tokens are rounded to the new scale
"""

import math

import torch

own = False

E_MIN = -64            # smallest exponent of a block
PAGE = 64              # tokens per cache page
BLOCK = 128            # columns (and weight rows) per scale of the projection
DEV = "cuda"


# ---- the cases -----------------------------------------------------------------------------------------------

def listed():
    return [
        # one sequence being decoded: the smallest product of a layer, bound by reading the weight
        {"name": "fp8 o, 1 token", "op": "fp8", "m": 1, "n": 4096, "k": 4096},
        # a few sequences on a ragged slice of a weight: odd row and column counts, tail blocks in both directions
        {"name": "fp8 ragged, 27 tokens", "op": "fp8", "m": 27, "n": 4093, "k": 2064},
        # the benchmark's tallest weight at its largest decode batch: between bandwidth and arithmetic
        {"name": "fp8 qkv_gate, 256 tokens", "op": "fp8", "m": 256, "n": 12288, "k": 4096},
        # a prompt through the same weight: bound by arithmetic
        {"name": "fp8 qkv_gate, 4096 tokens", "op": "fp8", "m": 4096, "n": 12288, "k": 4096},
        # one new token for each of 32 sequences, most of them in the middle of a page
        {"name": "append 32 x 1", "op": "append", "batch": 32, "new": 1, "ragged": False, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "interleaved": False, "scaling": "none", "past": 1500},
        # drafted tokens, up to 5 a sequence (some have none), interleaved pairs on half of each head
        {"name": "append drafts 45 x 0..5", "op": "append", "batch": 45, "new": 5, "ragged": True, "q_heads": 16, "kv_heads": 4, "dim": 64,
         "rot": 32, "interleaved": True, "scaling": "linear", "past": 700},
        # prompts: whole pages are written, positions far beyond the trained range
        {"name": "append prompts 3 x ..1500", "op": "append", "batch": 3, "new": 1500, "ragged": True, "q_heads": 32, "kv_heads": 16, "dim": 128,
         "rot": 128, "interleaved": False, "scaling": "yarn", "past": 60000},
        # one sequence, one token, a short history: latency
        {"name": "attend 1 x 300", "op": "attend", "batch": 1, "new": 1, "ragged": False, "q_heads": 32, "kv_heads": 8, "dim": 128, "ctx": 300,
         "window": 0, "gate": True},
        # a full decode batch with lengths from one token up: bound by reading the cache
        {"name": "attend 64 x ..4000", "op": "attend", "batch": 64, "new": 1, "ragged": True, "q_heads": 32, "kv_heads": 16, "dim": 128, "ctx": 4000,
         "window": 0, "gate": True},
        # two long documents: few rows, the long axis has to be split
        {"name": "attend 2 x 100000", "op": "attend", "batch": 2, "new": 1, "ragged": False, "q_heads": 32, "kv_heads": 4, "dim": 128, "ctx": 100000,
         "window": 0, "gate": False},
        # drafted tokens being checked, a sliding window, sequences without a token among them
        {"name": "attend drafts 21 x 0..4", "op": "attend", "batch": 21, "new": 4, "ragged": True, "q_heads": 16, "kv_heads": 4, "dim": 64, "ctx": 3001,
         "window": 1000, "gate": False},
        # a chunk of two prompts against what the cache holds of them: bound by arithmetic
        {"name": "attend chunk 2 x 512", "op": "attend", "batch": 2, "new": 512, "ragged": False, "q_heads": 32, "kv_heads": 8, "dim": 128, "ctx": 4096,
         "window": 0, "gate": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["fp8", "append", "attend", "attend"])
    if op == "fp8":
        m, n, k = _log(rng, 1, 4096), _log(rng, 128, 12288), 16 * _log(rng, 8, 512)
        if rng.random() < 0.5:
            n = max(16, n // 16 * 16)
        while m * n * k > 4096 * 12288 * 4096:
            m //= 2
        return {"op": op, "m": m, "n": n, "k": k}
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8, 16])
    heads = min(64, kv * rng.choice([1, 2, 4, 8]))
    if op == "append":
        new = rng.choice([1, rng.randint(2, 8), _log(rng, 9, 1500)])
        batch = max(1, min(_log(rng, 1, 128), 4096 // new))
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
        return {"op": op, "batch": batch, "new": new, "ragged": rng.random() < 0.6, "q_heads": heads, "kv_heads": kv, "dim": dim, "rot": rot,
                "interleaved": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "past": _log(rng, 1, 60000 // max(1, batch // 4))}
    new = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 512)])
    ctx = max(new, _log(rng, 1, 100000))
    batch = _log(rng, 1, 64)
    while batch > 1 and batch * ctx * kv * dim > 64 * 4000 * 16 * 128:
        batch = (batch + 1) // 2
    while new > 1 and (batch * new * ctx * heads * dim > 2 * 512 * 4096 * 32 * 128 or batch * new * ctx * heads > 1 << 29):
        new //= 2
    return {"op": op, "batch": batch, "new": new, "ragged": rng.random() < 0.6, "q_heads": heads, "kv_heads": kv, "dim": dim, "ctx": ctx,
            "window": rng.choice([0, 0, _log(rng, 1, max(2, ctx))]), "gate": rng.random() < 0.5}


# ---- number formats --------------------------------------------------------------------------------------------

def _power(byte):
    """2^(byte - 127) as FP32, from the exponent byte."""
    return (byte.to(torch.int32) << 23).view(torch.float32)


def _exponent_byte(amax):
    """The exponent byte of a block with this largest magnitude: 448 = 0.875 * 2^9."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(min=E_MIN) + 127


def _amax(x, dim):
    return torch.where(x.isfinite(), x.abs(), torch.zeros_like(x)).amax(dim)


def _codes(x, byte):
    """FP32 x as e4m3 codes under the exponent byte (broadcast)."""
    y = (x * _power(254 - byte)).clamp(-448.0, 448.0)
    return torch.where(x.isfinite(), y, torch.full_like(y, float("nan"))).to(torch.float8_e4m3fn)


def _blocks(x, size):
    """The last axis cut into blocks of `size`, the last one filled with zeros."""
    pad = -x.shape[-1] % size
    return torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, size))


# ---- inputs ----------------------------------------------------------------------------------------------------

def _inverse_frequencies(rot, scaling, base=10000.0, factor=4.0, trained=16384):
    i = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
    inv, amplitude = base ** (-2.0 * i / rot), 1.0
    if scaling == "linear":                     # positions divided by the factor
        inv = inv / factor
    elif scaling == "ntk":                      # a larger base: the slowest pair is slowed by the factor
        inv = (base * factor ** (rot / max(rot - 2, 1))) ** (-2.0 * i / rot)
    elif scaling == "yarn":                     # pairs that turn often keep their frequency, slow ones are slowed
        keep = ((trained * inv / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        inv, amplitude = inv * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1.0
    return inv, amplitude


def _lengths(case, total):
    """New tokens and total length of each sequence, the same for every seed of a case. A ragged batch has short ones,
    and sequences without a new token."""
    g = torch.Generator().manual_seed(total + 7)
    b, new = case["batch"], case["new"]
    q = torch.full((b,), new, dtype=torch.int64)
    length = torch.full((b,), total, dtype=torch.int64)
    if case["ragged"]:
        length = 1 + (torch.rand((b,), generator=g) * (total - 1) + 0.5).long()
        length[0] = total
        q = torch.randint(0 if new > 1 and b > 1 else 1, new + 1, (b,), generator=g)
        q[0] = new
        q = torch.minimum(q, length)
    cu = torch.zeros((b + 1,), dtype=torch.int64)
    cu[1:] = q.cumsum(0)
    return q, length, cu


def _cache(pages, kv, dim, gen):
    """A cache in use: every page holds quantised values, of this or an earlier sequence; heads differ in magnitude."""
    size = torch.exp(0.7 * torch.randn((pages, kv, 1, 1), generator=gen, device=DEV))
    k = torch.randn((pages, kv, PAGE, dim), generator=gen, device=DEV) * size
    kb = _exponent_byte(_amax(k.flatten(2), -1))
    k = _codes(k, kb[..., None, None])
    v = torch.randn((pages, kv, dim, PAGE), generator=gen, device=DEV) * size
    vb = _exponent_byte(_amax(v.flatten(2), -1))
    v = _codes(v, vb[..., None, None])
    return {"k": k, "v": v, "kb": kb.to(torch.uint8), "vb": vb.to(torch.uint8)}


def _paged(case, length, g, gen):
    """Page table over a shuffled pool (page 0 belongs to nobody) and the pool itself."""
    need = (length + PAGE - 1) // PAGE
    width = int(need.max())
    order = torch.randperm(int(need.sum()), generator=g) + 1
    table = torch.zeros((case["batch"], width), dtype=torch.int64)
    at = torch.arange(width)[None, :] < need[:, None]
    table[at] = order
    pool = _cache(int(need.sum()) + 1, case["kv_heads"], case["dim"], gen)
    pool["table"] = table.to(torch.int32).to(DEV)
    return pool


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    g = torch.Generator().manual_seed(seed)
    if case["op"] == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        w = 0.02 * torch.randn((n, k), generator=gen, device=DEV)
        tiles = _blocks(_blocks(w, BLOCK).permute(1, 2, 0), BLOCK).permute(2, 0, 3, 1)      # [N / 128, K / 128, 128, 128]
        byte = _exponent_byte(_amax(tiles.flatten(2), -1))
        w8 = _codes(w, byte.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k])
        x = torch.randn((m, k), generator=gen, device=DEV) * torch.exp(0.5 * torch.randn((1, k), generator=gen, device=DEV))
        return {"case": case, "x": x.to(torch.bfloat16), "w8": w8, "wb": byte.to(torch.uint8)}
    new, hq, hk, d = case["new"], case["q_heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        total = case["past"] + new
        q, length, cu = _lengths(case, total)
        m = int(cu[-1])
        s = _paged(case, length, g, gen)
        width = (hq + 2 * hk) * d + hq * d                                # q | k | v | gate: a projection's rows
        spread = torch.exp(0.7 * torch.randn((m, 1), generator=gen, device=DEV))
        s["qkv"] = (torch.randn((m, width), generator=gen, device=DEV) * spread).to(torch.bfloat16)
        inv, amplitude = _inverse_frequencies(case["rot"], case["scaling"])
        angle = torch.arange(s["table"].shape[1] * PAGE, dtype=torch.float64, device=DEV)[:, None] * inv
        s["cos_sin"] = (amplitude * torch.stack([angle.cos(), angle.sin()], -1)).float()
    else:
        q, length, cu = _lengths(case, case["ctx"])
        m = int(cu[-1])
        s = _paged(case, length, g, gen)
        s["q"] = torch.randn((m, hq, d), generator=gen, device=DEV).to(torch.bfloat16)
        s["gate"] = torch.randn((m, hq * d), generator=gen, device=DEV).to(torch.bfloat16) if case["gate"] else None
    s["case"] = case
    s["length"], s["cu"] = length.to(torch.int32).to(DEV), cu.to(torch.int32).to(DEV)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def _project(s):
    x, (n, k) = s["x"].float(), s["w8"].shape
    xb = _blocks(x, BLOCK)
    byte = _exponent_byte(_amax(xb, -1))[..., None]
    xq = (_codes(xb, byte).float() * _power(byte)).flatten(1)[:, :k]
    scale = _power(s["wb"]).repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return (xq @ (s["w8"].float() * scale).T).to(torch.bfloat16)


def _tokens(s):
    """For each new token its sequence and its position (below zero: a token that is not in the sequence)."""
    cu, length = s["cu"].long(), s["length"].long()
    m = (s["qkv"] if "qkv" in s else s["q"]).shape[0]
    t = torch.arange(m, device=DEV)
    seq = torch.searchsorted(cu[1:], t, right=True)
    return seq, length[seq] - cu[seq + 1] + t


def _rotate(x, cs, interleaved):
    rot = 2 * cs.shape[-2]
    c, n = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2 : rot])
    ya, yb = a * c - b * n, b * c + a * n
    y = torch.stack([ya, yb], -1).flatten(-2) if interleaved else torch.cat([ya, yb], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _append_half(pool, byte, new, page, slot, head, touched, first, transposed):
    """Writes `new` [m, heads, dim] into a pool of codes at (page, slot): scales of the touched pages first, then the
    codes of their earlier tokens under the new scale, then the new tokens. Returns the values the pool then holds."""
    a = _amax(new, -1)                                                               # [m, heads]
    at = page[:, None] * byte.shape[1] + head
    top = torch.zeros(byte.numel(), device=DEV).scatter_reduce_(0, at.flatten(), a.flatten(), "amax")
    fresh = _exponent_byte(top).view_as(byte)
    old = byte.to(torch.int32)
    kept = first[:, None] > 0                                                        # [pages, 1]: the page holds earlier tokens
    raised = torch.where(touched[:, None], torch.where(kept, torch.maximum(fresh, old), fresh), old)
    pages = pool["pages"]                                                            # the pages that new tokens fall into
    data = pool["codes"]
    was = data[pages].view(torch.float8_e4m3fn).float() * _power(old[pages])[..., None, None]
    earlier = (torch.arange(PAGE, device=DEV) < first[pages][:, None])[:, None]      # [pages, 1, token]
    earlier = earlier[:, :, None] if transposed else earlier[..., None]
    earlier = earlier & touched[pages][:, None, None, None]
    data[pages] = torch.where(earlier, _codes(was, raised[pages][..., None, None]).view(torch.uint8), data[pages])
    byte.copy_(raised.to(torch.uint8))
    q = _codes(new, raised[page][..., None])
    if transposed:
        data[page[:, None], head[None, :], :, slot[:, None]] = q.view(torch.uint8)
    else:
        data[page[:, None], head[None, :], slot[:, None]] = q.view(torch.uint8)
    return (q.float() * _power(raised[page])[..., None]).to(torch.bfloat16)


def _append(s):
    c = s["case"]
    hq, hk, d = c["q_heads"], c["kv_heads"], c["dim"]
    seq, pos = _tokens(s)
    page, slot = s["table"].long()[seq, pos // PAGE], pos % PAGE
    x = s["qkv"][:, : (hq + 2 * hk) * d].float().unflatten(1, (-1, d))
    rotated = _rotate(x[:, : hq + hk], s["cos_sin"][pos], c["interleaved"])
    first = torch.full((s["kb"].shape[0],), PAGE, device=DEV).scatter_reduce_(0, page, slot, "amin")
    touched = first < PAGE
    reach = (c["new"] + PAGE - 2) // PAGE + 1                                        # pages that a sequence's new tokens can fall into
    start = (s["length"].long() - s["cu"].long().diff()) // PAGE
    span = (start[:, None] + torch.arange(reach, device=DEV)).clamp(max=s["table"].shape[1] - 1)
    pages = s["table"].long().gather(1, span).flatten()
    head = torch.arange(hk, device=DEV)
    out = [rotated[:, :hq].to(torch.bfloat16)]
    for name, new, transposed in (("k", rotated[:, hq:], False), ("v", x[:, hq + hk :], True)):
        pool = {"codes": s[name].view(torch.uint8), "pages": pages}
        out.append(_append_half(pool, s[name + "b"], new, page, slot, head, touched, first, transposed))
    return out + [s["k"], s["v"], s["kb"], s["vb"]]


def _attend(s):
    c = s["case"]
    hq, hk, d, new = c["q_heads"], c["kv_heads"], c["dim"], c["new"]
    b, table = c["batch"], s["table"].long()
    k = (s["k"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * _power(s["kb"][table])[..., None, None]).transpose(1, 2).flatten(2, 3)
    v = (s["v"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * _power(s["vb"][table])[..., None, None]).permute(0, 2, 1, 4, 3).flatten(2, 3)
    cu, length = s["cu"].long(), s["length"].long()
    t = cu[:-1, None] + torch.arange(new, device=DEV)                                # the tokens of each sequence, [b, new]
    live = t < cu[1:, None]
    q = s["q"][t.clamp(max=s["q"].shape[0] - 1)].float().view(b, new, hk, hq // hk, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = (q @ k.transpose(2, 3)).unflatten(2, (hq // hk, new)) / math.sqrt(d)     # [b, hk, group, new, tokens]
    pos = length[:, None] - cu[1:, None] + t                                         # [b, new]
    j = torch.arange(k.shape[2], device=DEV)
    seen = (j <= pos[..., None]) & (j < length[:, None, None])
    if c["window"]:
        seen = seen & (j > pos[..., None] - c["window"])
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top.isfinite(), top, torch.zeros_like(top)))
    o = (p.flatten(2, 3) @ v).unflatten(2, (hq // hk, new)) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).flatten(2)[live]                                    # [m, heads * dim], in the tokens' order
    if s["gate"] is not None:
        o = o * torch.sigmoid(s["gate"].float())
    return o.to(torch.bfloat16)


def _run_own(s):
    from llm_inference_engine_b200 import cache8, fp8

    c = s["case"]
    if c["op"] == "fp8":
        return fp8.linear(s["x"], s["w8"], s["wb"])
    cache = cache8.Cache8(s["k"], s["v"], s["kb"], s["vb"])
    cu = None if c["new"] == 1 and not c["ragged"] else s["cu"]
    if c["op"] == "append":
        q, k, v = cache8.rope_append(s["qkv"], cache, s["cos_sin"], s["table"], s["length"], q_heads=c["q_heads"], cu_q=cu, max_q=c["new"],
                                     interleaved=c["interleaved"], values=True)
        return [q, k, v, s["k"], s["v"], s["kb"], s["vb"]]
    return cache8.attention(s["q"], cache, s["table"], s["length"], cu_q=cu, max_q=c["new"], window=c["window"], gate=s["gate"])


def run(state):
    if own:
        return _run_own(state)
    return {"fp8": _project, "append": _append, "attend": _attend}[state["case"]["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------

def work(case):
    if case["op"] == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k + -(-n // BLOCK) * -(-k // BLOCK) + 2 * m * k + 2 * m * n, "flops": 2 * m * n * k}
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    q, length, cu = _lengths(case, case["past"] + case["new"] if case["op"] == "append" else case["ctx"])
    m = int(cu[-1])
    if case["op"] == "append":
        # q, k, v read; q and the values written in BF16, the codes in 8 bits; the rotary table's rows
        return {"bytes": m * ((hq + 2 * hk) * d * 4 + 2 * hk * d + case["rot"] * 4) + 8 * case["batch"], "flops": 3 * m * (hq + hk) * case["rot"]}
    seen, pairs = 0, 0
    for n, total in zip(q.tolist(), length.tolist()):
        if n:
            w = case["window"] or total
            seen += min(total, w + n - 1)
            pairs += sum(min(w, total - n + i + 1) for i in range(n))
    return {"bytes": seen * hk * d * 2 + m * hq * d * (6 if case["gate"] else 4) + 8 * case["batch"], "flops": 4 * pairs * hq * d}


# ---- the same in 64 bits, written from the definitions ---------------------------------------------------------

def _value(code, byte):
    return code.view(torch.float8_e4m3fn).double() * torch.exp2(byte.double() - 127.0)


def _quantised64(x, dims):
    """x in 64 bits rounded to the format over blocks that span `dims`; the values that the codes stand for."""
    a = x.abs().amax(dims, keepdim=True)
    e = torch.where(a > 0, torch.ceil(torch.log2(a.clamp(min=1e-300) / 448.0)), torch.full_like(a, E_MIN)).clamp(min=E_MIN)
    # log2 may land beside a whole number: settle it by the values themselves
    e = torch.where(a > 448.0 * torch.exp2(e), e + 1, e)
    e = torch.where((a <= 448.0 * torch.exp2(e - 1)) & (e > E_MIN), e - 1, e)
    y = x / torch.exp2(e)
    step = torch.exp2((torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))).clamp(max=8) - 3.0)
    return torch.round(y / step) * step * torch.exp2(e), e


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "fp8":
        x, w = s["x"].double(), s["w8"].double()
        n, k = w.shape
        out = torch.zeros((x.shape[0], n), dtype=torch.float64, device=DEV)
        for c in range(0, k, BLOCK):
            xq, _ = _quantised64(x[:, c : c + BLOCK], (1,))
            rows = torch.exp2(s["wb"][:, c // BLOCK].double() - 127.0).repeat_interleave(BLOCK)[:n]
            out += xq @ (w[:, c : c + BLOCK] * rows[:, None]).T
        return out
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    cu, length, table = s["cu"].tolist(), s["length"].tolist(), s["table"].tolist()
    if case["op"] == "append":
        m, rot = s["qkv"].shape[0], case["rot"]
        inv, amplitude = _inverse_frequencies(rot, case["scaling"])
        x = s["qkv"].double()
        pos = torch.cat([torch.arange(n - (b - a), n, device=DEV) for a, b, n in zip(cu, cu[1:], length)]).double()
        z = amplitude * torch.polar(torch.ones((m, 1, rot // 2), dtype=torch.float64, device=DEV), pos[:, None, None] * inv)
        heads = x[:, : (hq + hk) * d].reshape(m, hq + hk, d)
        pairs = heads[..., :rot].reshape(m, -1, rot // 2, 2) if case["interleaved"] else heads[..., :rot].reshape(m, -1, 2, rot // 2).transpose(2, 3)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
        turned = (turned if case["interleaved"] else turned.transpose(2, 3)).reshape(m, hq + hk, rot)
        y = torch.cat([turned, heads[..., rot:]], -1)
        out = {}
        for name, new in (("k", y[:, hq:]), ("v", x[:, (hq + hk) * d : (hq + 2 * hk) * d].reshape(m, hk, d))):
            held = torch.empty_like(new)
            for row, a, b, n in zip(table, cu, cu[1:], length):
                t = a
                while t < b:
                    p = n - b + t
                    end = min(b, t + PAGE - p % PAGE)
                    part = new[t:end].transpose(0, 1)                                    # [heads, tokens, dim]
                    _, e = _quantised64(part, (1, 2))
                    if p % PAGE:
                        e = torch.maximum(e, s[name + "b"][row[p // PAGE]].double()[:, None, None] - 127.0)
                    y8 = part / torch.exp2(e)
                    step = torch.exp2(torch.floor(torch.log2(y8.abs().clamp(min=2.0 ** -6))).clamp(max=8) - 3.0)
                    held[t:end] = (torch.round(y8 / step) * step * torch.exp2(e)).transpose(0, 1)
                    t = end
            out[name] = held
        return [y[:, :hq], out["k"], out["v"], None, None, None, None]
    out = torch.zeros((s["q"].shape[0], hq, d), dtype=torch.float64, device=DEV)
    for i, n in enumerate(length):
        new = cu[i + 1] - cu[i]
        if not new:
            continue
        lo = max(0, n - new - case["window"] + 1) // PAGE if case["window"] else 0
        pages = s["table"][i, lo : (n + PAGE - 1) // PAGE].long()
        j = torch.arange(lo * PAGE, lo * PAGE + len(pages) * PAGE, device=DEV)
        pos = torch.arange(n - new, n, device=DEV)[:, None]
        hidden = (j > pos) | (j <= pos - case["window"] if case["window"] else j < 0)
        for h in range(hk):
            k = _value(s["k"].view(torch.uint8)[pages, h], s["kb"][pages, h][:, None, None]).reshape(-1, d)
            v = _value(s["v"].view(torch.uint8)[pages, h], s["vb"][pages, h][:, None, None]).transpose(1, 2).reshape(-1, d)
            for a in range(h * (hq // hk), (h + 1) * (hq // hk)):
                score = s["q"][cu[i] : cu[i + 1], a].double() @ k.T / math.sqrt(d)
                out[cu[i] : cu[i + 1], a] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v
    out = out.flatten(1)
    return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())
