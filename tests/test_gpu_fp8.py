"""The 8-bit projection (fp8.quantize, fp8.linear, kernel_fn_fp8) against its definition in 64 bits.

Codes and exponents have to be the ones the format defines, bit for bit. The product's codes and scales are exact in
FP32, so a result is off by its rounding to BF16 (2^-8 relative) and by the FP32 sums: at most one rounding or
truncation (2^-23) of the sum of magnitudes S per added column, K 2^-23 S."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def fp8():
    from llm_inference_engine_b200 import fp8

    return fp8


def quantised64(x: torch.Tensor):
    """x [m, K] per token and 128 columns, in 64 bits: the values the codes stand for, and the exponents. Written from
    the definition: the smallest e >= -64 with amax <= 448 * 2^e; codes are multiples of 2^(max(floor(log2 |y|), -6) - 3)."""
    m, k = x.shape
    y = torch.nn.functional.pad(x.double(), (0, -k % 128)).view(m, -1, 128)
    a = torch.where(y.isfinite(), y.abs(), torch.zeros_like(y)).amax(-1, keepdim=True)
    e = torch.full_like(a, -64.0)
    while bool((a > 448.0 * torch.exp2(e)).any()):
        e = torch.where(a > 448.0 * torch.exp2(e), e + 1, e)
    z = y / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))).clamp(max=8.0) - 3.0)
    q = torch.round(z / step) * step * torch.exp2(e)
    q = torch.where(y.isfinite(), q, torch.full_like(q, float("nan")))
    return q.flatten(1)[:, :k], e[..., 0]


def check_linear(out, x, w_values):
    xq, _ = quantised64(x)
    want = xq @ w_values.double().T
    room = 2.0 ** -8 * want.abs() + x.shape[1] * 2.0 ** -23 * (xq.abs() @ w_values.double().abs().T)
    assert out.dtype == torch.bfloat16 and out.shape == want.shape
    bad = ((out.double() - want).abs() > room).sum().item()
    assert bad == 0, f"{bad} of {out.numel()} results are outside the rounding"


def inputs(m, n, k, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn((m, k), generator=g, device=DEV) * torch.exp(torch.randn((1, k), generator=g, device=DEV))
    w = 0.02 * torch.randn((n, k), generator=g, device=DEV)
    return x.bfloat16(), w


@pytest.mark.parametrize("m,k", [(1, 16), (3, 4096), (9, 1040), (130, 2064), (1, 12304)])
def test_quantize_is_the_format_bit_for_bit(fp8, m, k):
    x, _ = inputs(m, 1, k, m + k)
    x[0, : min(k, 128)] = 0                                   # a block of zeros takes the smallest exponent
    if k > 256:
        x[-1, 128:256] = 0
        x[-1, 130] = 2.0 ** -100                              # far below the smallest scale
    q, e = fp8.quantize(x)
    want, we = quantised64(x)
    assert torch.equal(e.double() - 127.0, we)
    scale = torch.exp2(we).repeat_interleave(128, 1)[:, :k]
    assert torch.equal(q.double() * scale, want)


def test_exponents_at_their_borders_and_what_is_not_finite(fp8):
    x = torch.zeros((6, 128), device=DEV)
    x[0, 5], x[1, 5], x[2, 5], x[3, 5] = 448.0, 450.0, 3.0e38, 1.75 * 2.0 ** -40
    x[4, 5], x[4, 6] = float("inf"), 7.0
    x[5, 5], x[5, 7] = float("nan"), -float("inf")
    x = x.bfloat16()
    q, e = fp8.quantize(x)
    want, we = quantised64(x)
    assert torch.equal(e.double() - 127.0, we)
    got = q.double() * torch.exp2(we)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~got.isnan()], want[~want.isnan()])
    assert got[4, 5].isnan() and got[4, 6] == 7.0


def test_weight_codes_round_trip(fp8):
    _, w = inputs(1, 300, 1040, 5)
    w8, we = fp8.quantize_weight(w)
    assert w8.shape == (300, 1040) and we.shape == (3, 9) and we.dtype == torch.uint8
    back = fp8.dequantize_weight(w8, we)
    assert bool(((back - w).abs() <= 2.0 ** -4 * w.abs() + 2.0 ** -10 * torch.exp2(we.float() - 127).repeat_interleave(128, 0)[:300].repeat_interleave(128, 1)[:, :1040]).all())
    again, again_e = fp8.quantize_weight(back)
    assert torch.equal(again.view(torch.uint8), w8.view(torch.uint8)) and torch.equal(again_e, we)
    cpu8, cpue = fp8.quantize_weight(w.cpu())
    assert torch.equal(cpu8.view(torch.uint8), w8.cpu().view(torch.uint8)) and torch.equal(cpue, we.cpu())


SHAPES = [(1, 4096, 4096), (2, 1024, 4096), (8, 4096, 1024), (5, 1000, 1040), (3, 7, 16), (16, 4096, 4096), (9, 777, 8192), (13, 130, 6160),
          (4, 12288, 4096), (8, 100, 8192), (16, 64, 144), (17, 4096, 4096), (27, 4093, 2064), (33, 333, 12304), (64, 2304, 4096), (100, 129, 272),
          (128, 4096, 1024), (256, 1024, 4096), (1, 333, 12304), (300, 515, 528), (1000, 640, 1056), (513, 4100, 4096)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_matches_64_bits(fp8, m, n, k):
    x, w = inputs(m, n, k, 7 * m + n + k)
    w8, we = fp8.quantize_weight(w)
    values = fp8.dequantize_weight(w8, we)
    check_linear(fp8.linear(x, w8, we), x, values)
    check_linear(fp8.linear(fp8.quantize(x), w8, we), x, values)


@pytest.mark.parametrize("m", [1, 7, 20, 200])
def test_blocks_of_different_scale_meet(fp8, m):
    """Scales that differ by 2^30 between neighbouring blocks of x and of W, zero blocks, the largest codes."""
    x, w = inputs(m, 400, 1040, 50 + m)
    x = (x.float() * torch.exp2(torch.randint(-15, 16, (m, 9), device=DEV).float()).repeat_interleave(128, 1)[:, :1040]).bfloat16()
    w = w * torch.exp2(torch.randint(-15, 16, (4, 9), device=DEV).float()).repeat_interleave(128, 0)[:400].repeat_interleave(128, 1)[:, :1040]
    x[:, 256:384] = 0
    w[128:256, 512:640] = 0
    x[:, 0] = x[:, :128].abs().amax(1) * 1.5
    w8, we = fp8.quantize_weight(w)
    check_linear(fp8.linear(x, w8, we), x, fp8.dequantize_weight(w8, we))


@pytest.mark.parametrize("m", [1, 12, 40, 300])
def test_a_value_that_is_not_finite_spoils_its_token_only(fp8, m):
    x, w = inputs(m, 520, 1040, 60 + m)
    x[0, 700] = float("inf")
    w8, we = fp8.quantize_weight(w)
    out = fp8.linear(x, w8, we)
    assert bool(out[0].isnan().all()) and bool(out[1:].isfinite().all())
    if m > 1:
        check_linear(out[1:], x[1:], fp8.dequantize_weight(w8, we))


@pytest.mark.parametrize("m", [1, 9, 70, 257])
def test_strides_out_and_neighbours(fp8, m):
    """x as a slice of wider rows, x misaligned (copied), out as a slice whose neighbours stay as they were."""
    x, w = inputs(m, 515, 528, 70 + m)
    w8, we = fp8.quantize_weight(w)
    want = fp8.linear(x, w8, we)
    wide = torch.randn((m, 700), device=DEV).bfloat16()
    wide[:, 8 : 8 + 528] = x
    assert torch.equal(fp8.linear(wide[:, 8:536], w8, we), want)
    odd = torch.randn((m, 533), device=DEV).bfloat16()
    odd[:, 3 : 3 + 528] = x
    assert torch.equal(fp8.linear(odd[:, 3:531], w8, we), want)
    assert torch.equal(fp8.linear(x.T.contiguous().T, w8, we), want)
    for width, at in ((600, 0), (521, 3), (528, 8)):
        big = torch.full((m + 2, width + at), 7.0, device=DEV, dtype=torch.bfloat16)
        got = fp8.linear(x, w8, we, out=big[1:-1, at:])
        assert got.data_ptr() == big[1:-1, at:].data_ptr() and torch.equal(got[:, :515], want)
        assert bool((big[0] == 7).all()) and bool((big[-1] == 7).all()) and bool((big[:, :at] == 7).all()) and bool((big[:, at + 515 :] == 7).all())


def test_replay_streams_and_same_bits(fp8):
    """Captured on one stream and replayed with x rewritten, two graphs replayed at once on two streams, eager calls on a
    side stream: the bits of the eager call each time."""
    _, w = inputs(1, 1000, 1040, 80)
    w8, we = fp8.quantize_weight(w)
    torch.cuda.synchronize(DEV)
    for m in (1, 16, 17, 128, 300):
        xs = [inputs(m, 1, 1040, 90 + i)[0] for i in range(3)]
        want = [fp8.linear(x, w8, we) for x in xs]
        assert all(torch.equal(fp8.linear(x, w8, we), y) for x, y in zip(xs, want))
        graphs, bufs, outs = [], [], []
        for i in range(2):
            bufs.append(xs[i].clone())
            side = torch.cuda.Stream(DEV)
            side.wait_stream(torch.cuda.current_stream(DEV))
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(fp8.linear(bufs[i], w8, we))
            graphs.append((g, side))
        for turn in range(20):
            torch.cuda.synchronize(DEV)
            for (g, side), b in zip(graphs, bufs):
                with torch.cuda.stream(side):
                    b.copy_(xs[(turn + len(bufs)) % 3] if turn % 2 else xs[turn % 3])
                    g.replay()
            torch.cuda.synchronize(DEV)
            i = (turn + 2) % 3 if turn % 2 else turn % 3
            assert torch.equal(outs[0], want[i]) and torch.equal(outs[1], want[i]), (m, turn)


def test_behind_the_layer_names(fp8):
    from llm_inference_engine_b200 import muse_bf16_proj as proj

    g = torch.Generator(device=DEV).manual_seed(3)
    weights = {"o": 0.02 * torch.randn((512, 1024), generator=g, device=DEV), "unpooler": 0.02 * torch.randn((640, 256), generator=g, device=DEV)}
    weights = {k: v.bfloat16() for k, v in weights.items()}
    weights["router"] = torch.randn((64, 1024), generator=g, device=DEV)
    state = proj.prepare(weights, warmup=False)
    x = torch.randn((6, 256), generator=g, device=DEV).bfloat16()
    cfg = {"layer": "unpooler", "m": 6, "n": 200, "k": 256}
    with pytest.raises(KeyError, match="prepare_fp8"):
        proj.kernel_fn_fp8({"x": x, "config": cfg}, state)
    proj.prepare_fp8(state)
    assert set(state["_fp8"]) == {"o", "unpooler"}
    w8, we = fp8.quantize_weight(weights["unpooler"])
    got = proj.kernel_fn_fp8({"x": x, "config": cfg}, state)
    check_linear(got, x, fp8.dequantize_weight(w8, we)[:200])
    with pytest.raises(TypeError):
        proj.prepare_fp8(state, ["router"])
    with pytest.raises(KeyError):
        proj.prepare_fp8(state, ["pooler"])
    with pytest.raises(ValueError):
        proj.kernel_fn_fp8({"x": x, "config": dict(cfg, n=641)}, state)


def test_refusals(fp8):
    x, w = inputs(4, 100, 272, 1)
    w8, we = fp8.quantize_weight(w)
    for bad in (x.float(), x[0]):
        with pytest.raises(TypeError):
            fp8.linear(bad, w8, we)
        with pytest.raises(TypeError):
            fp8.quantize(bad)
    for args in ((x[:, :256], w8, we), (x, w8, we[:, :2]), (x, w8.view(torch.uint8).T.contiguous().T.view(torch.float8_e4m3fn), we),
                 (x[:0], w8, we), (x[:, :264].contiguous(), w8[:, :264].contiguous(), we)):
        with pytest.raises(ValueError):
            fp8.linear(*args)
    with pytest.raises(TypeError):
        fp8.linear(x, w8.view(torch.uint8), we)
    with pytest.raises(TypeError):
        fp8.linear(x, w8, we.int())
    with pytest.raises(ValueError):
        fp8.linear(x, w8, we, out=torch.empty((4, 99), device=DEV, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        fp8.linear(x, w8, we, out=torch.empty((4, 100), device=DEV))
    with pytest.raises(ValueError):
        fp8.quantize(x[:, :40].contiguous())
    with pytest.raises(RuntimeError, match="CUDA device only"):
        fp8.linear(x.cpu(), w8.cpu(), we.cpu())


@pytest.mark.parametrize("m", [1, 8, 20, 200])
def test_scales_whose_product_leaves_fp32(fp8, m):
    """A block of x near 2^104 against a block of W near 2^46: the two exponents add up to 133, more than FP32's scale factors
    reach, while products of its small codes, and zeros, are inside FP32. Rows beyond FP32 are infinite."""
    x, w = inputs(m, 256, 272, 90 + m)
    x[:, :128], w[:128, :128] = 0, 0
    x[:, 0] = 2.0**104          # met by zeros of W, but in the last rows of its block
    x[:, 1:9] = 2.0**87         # small codes of the same block
    w[1:120, 9] = 2.0**46       # met by zeros of x
    w[1:100, 1:9] = 2.0**29     # small codes of the same block
    w[120:128, 0] = 2.0**46
    w8, we = fp8.quantize_weight(w)
    _, xe = fp8.quantize(x)
    assert int(we[0, 0]) + int(xe[0, 0]) - 254 >= 128
    values = fp8.dequantize_weight(w8, we).double()
    want = quantised64(x)[0] @ values.T
    out = fp8.linear(x, w8, we)
    assert bool((want[:, 120:128] > 3.5e38).all()) and bool(out[:, 120:128].isinf().all())
    assert bool((want[:, 1:100] > 1e34).all()) and bool((want[:, 1:120].abs() < 3e38).all())
    rows = torch.cat([torch.arange(120), torch.arange(128, 256)]).to(DEV)
    room = 2.0**-8 * want.abs() + 272 * 2.0**-23 * (quantised64(x)[0].abs() @ values.abs().T)
    assert bool(((out.double() - want).abs() <= room)[:, rows].all()), (out[0, :4], want[0, :4])
