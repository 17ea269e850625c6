"""The MXFP8 product with its epilogue against the formula in 64 bits.

Whole-number inputs (codes of small whole numbers, scales of 1/2, 1 and 2): every product and every sum is a multiple of 1/4 below 2^22,
so fp32 holds it exactly in any order and the result has to be the formula's, rounded once, bit for bit. Other inputs: products of
two E4M3 values are exact; K - 1 additions that lose at most one unit in the last place each (2^-23) leave the sum within K * 2^-23 of
the sum of the absolute products, GAIN times that behind an activation; its own arithmetic adds 2^-16 relative; bf16 adds half a step, 2^-8."""
import math
import zlib

import pytest
import torch

from tests.test_gpu_add_rmsnorm import check_codes, mxfp8_of

pytestmark = pytest.mark.gpu

GAIN = 1.2  # the steepest slope of silu (1.0998) and of the two gelus (1.13)
ARITH = 2.0 ** -16


@pytest.fixture(scope="module")
def P():
    from amd_kernels_b200.moe import mxfp4_h6144_i768_e128_top4
    return mxfp4_h6144_i768_e128_top4


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    from amd_kernels_b200.moe.mxfp4_h6144_i768_e128_top4 import chain
    assert chain.last_status() == 0


def gen_of(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def whole(gen, m, k):
    """codes of -2 .. 2 and scales of 1/2, 1, 2, as bytes"""
    codes = torch.randint(-2, 3, (m, k), generator=gen, device="cuda").float().to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, torch.randint(126, 129, (m, k // 32), generator=gen, device="cuda", dtype=torch.uint8)


def real(gen, m, k, scale=1.0):
    x = torch.randn((m, k), generator=gen, device="cuda") * scale * torch.exp(0.5 * torch.randn(k, generator=gen, device="cuda"))
    byte = mxfp8_of(x.double(), 1)
    codes = (x.double() / torch.exp2(byte - 127).repeat_interleave(32, -1)).float().to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, byte.to(torch.uint8)


def values(codes, scales):
    return codes.view(torch.float8_e4m3fn).double() * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def activation(p, act):
    if act == "relu":
        return p.clamp_min(0)
    if act == "silu":
        return p * torch.sigmoid(p)
    if act == "gelu":
        return p * torch.special.ndtr(p)
    if act == "gelu_tanh":
        return p * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (p + 0.044715 * p ** 3))
    if act == "swiglu":
        g, u = p.chunk(2, -1)
        return g * torch.sigmoid(g) * u
    if act == "swiglu_oai":
        g, u = p.chunk(2, -1)
        g, u = g.clamp_max(7), u.clamp(-7, 7)
        return g * torch.sigmoid(1.702 * g) * (u + 1)
    return p


def formula(x, w, bias=None, act=None, residual=None):
    """(y, the bound on its fp32 error) in 64 bits"""
    xv, wv = values(*x), values(*w)
    p = xv @ wv.t()
    mass = xv.abs() @ wv.abs().t()
    if bias is not None:
        p, mass = p + bias.double(), mass + bias.double().abs()
    slack = mass * xv.shape[1] * 2.0 ** -23
    y = activation(p, act)
    if act is not None and act.startswith("swiglu"):
        (g, u), (sg, su) = p.chunk(2, -1), slack.chunk(2, -1)
        lin = (u.clamp(-7, 7) + 1).abs() if act == "swiglu_oai" else u.abs()  # y = a(g) * lin, |a(g)| <= |g| + 0.3, slope of a below GAIN
        slack = GAIN * sg * (lin + su) + (g.abs() + 0.3) * su
    elif act is not None:
        slack = GAIN * slack
    slack = slack + ARITH * y.abs()
    if residual is not None:
        y, slack = y + residual.double(), slack + 2.0 ** -24 * (y.abs() + residual.double().abs())
    return y, slack


SHAPES = [(1, 32, 8), (1, 6144, 4096), (2, 96, 40), (7, 128, 128), (16, 160, 136), (17, 512, 256), (33, 800, 264), (64, 2048, 1000),
          (65, 544, 96), (100, 6144, 512), (128, 256, 2048), (129, 1056, 392), (200, 4096, 128), (256, 128, 256), (257, 96, 264),
          (300, 2080, 640), (511, 512, 1032), (640, 288, 8), (777, 1536, 1544), (1025, 128, 4096), (1500, 4064, 768), (2100, 800, 2600)]


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_whole_numbers_bit_for_bit(P, m, k, n):
    gen = gen_of(m, k, n)
    x, w = whole(gen, m, k), whole(gen, n, k)
    bias = torch.randint(-8, 9, (n,), generator=gen, device="cuda").float()
    res = torch.randint(-64, 65, (m, n), generator=gen, device="cuda").bfloat16()
    weights = P.LinearWeights.from_row_major(*w, bias)
    p = values(*x) @ values(*w).t() + bias.double()
    y = P.mxfp8_linear(x, weights)
    assert torch.equal(y, p.float().bfloat16())
    assert torch.equal(P.mxfp8_linear(x, weights, activation="relu", residual=res), (p.clamp_min(0) + res.double()).float().bfloat16())
    assert torch.equal(P.mxfp8_linear(x, P.LinearWeights.from_row_major(*w)), (p - bias.double()).float().bfloat16())
    if n % 32 == 0:
        codes, scales = P.mxfp8_linear(x, weights, mxfp8_out=True)
        byte = mxfp8_of(p, 1)
        assert torch.equal(scales.double(), byte)
        want = (p / torch.exp2(byte - 127).repeat_interleave(32, -1)).float().to(torch.float8_e4m3fn)
        assert torch.equal(codes.view(torch.float8_e4m3fn).float(), want.float())


@pytest.mark.parametrize("m,k,n", [(1, 6144, 1024), (5, 800, 200), (48, 2048, 384), (130, 4096, 640), (333, 6144, 512), (1300, 1056, 776)])
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh"])
def test_activations_against_the_formula(P, m, k, n, act):
    gen = gen_of(m, k, n, act)
    x, w = real(gen, m, k), real(gen, n, k, 1.5 / math.sqrt(k))
    bias = 0.5 * torch.randn(n, generator=gen, device="cuda")
    res = torch.randn((m, n), generator=gen, device="cuda").bfloat16()
    weights = P.LinearWeights.from_row_major(*w, bias)
    for residual in (None, res):
        y, slack = formula(x, w, bias, act, residual)
        got = P.mxfp8_linear(x, weights, activation=act, residual=residual).double()
        assert bool(((got - y).abs() <= 2.0 ** -8 * y.abs() + 1.01 * slack).all())
        assert float((got - y).norm() / y.norm()) < 2.0 ** -8
    if n % 32 == 0:
        y, slack = formula(x, w, bias, act)
        check_codes(*P.mxfp8_linear(x, weights, activation=act, mxfp8_out=True), y, 1, 0.0, slack)


@pytest.mark.parametrize("m,k,n", [(1, 6144, 768), (3, 96, 32), (31, 512, 96), (120, 6144, 544), (150, 800, 160), (400, 2048, 512), (1111, 544, 1056)])
@pytest.mark.parametrize("act", ["swiglu", "swiglu_oai"])
def test_gated_against_the_formula(P, m, k, n, act):
    gen = gen_of(m, k, n, act)
    x, w = real(gen, m, k), real(gen, 2 * n, k, 2.0 / math.sqrt(k))
    bias = 0.5 * torch.randn(2 * n, generator=gen, device="cuda")
    weights = P.LinearWeights.from_row_major(*w, bias.bfloat16(), gated=True)
    assert weights.n == n
    y, slack = formula(x, w, bias.bfloat16(), act)
    got = P.mxfp8_linear(x, weights, activation=act).double()
    assert bool(((got - y).abs() <= 2.0 ** -8 * y.abs() + 1.01 * slack).all())
    codes, scales = P.mxfp8_linear(x, weights, activation=act, mxfp8_out=True)
    check_codes(codes, scales, y, 1, 0.0, slack)
    res = torch.randn((m, n), generator=gen, device="cuda").bfloat16()
    y, slack = formula(x, w, bias.bfloat16(), act, res)
    got = P.mxfp8_linear(x, weights, activation=act, residual=res).double()
    assert bool(((got - y).abs() <= 2.0 ** -8 * y.abs() + 1.01 * slack).all())


@pytest.mark.parametrize("m,k,n", [(1, 800, 96), (37, 544, 160), (200, 288, 640), (1000, 160, 416), (2200, 288, 4160)])
@pytest.mark.parametrize("act", [None, "silu", "gelu", "swiglu", "swiglu_oai"])
def test_mxfp8_result_with_a_residual(P, m, k, n, act):
    """The block's scale is that of the sum with the residual; codes that begin at 16 bytes of a sector, scales at any byte."""
    gen = gen_of(m, k, n, act, "mx")
    gated = act is not None and act.startswith("swiglu")
    rows = 2 * n if gated else n
    x, w = real(gen, m, k), real(gen, rows, k, 1.5 / math.sqrt(k))
    bias = 0.5 * torch.randn(rows, generator=gen, device="cuda")
    res = (3 * torch.randn((m, n), generator=gen, device="cuda")).bfloat16()
    weights = P.LinearWeights.from_row_major(*w, bias, gated=gated)
    y, slack = formula(x, w, bias, act, res)
    codes, scales = P.mxfp8_linear(x, weights, activation=act, residual=res, mxfp8_out=True)
    check_codes(codes, scales, y, 1, 0.0, slack)
    room, sroom = (torch.full((size + 48,), 93, dtype=torch.uint8, device="cuda") for size in (m * n, m * (n // 32)))
    out = room[16:m * n + 16].view(m, n), sroom[3:m * (n // 32) + 3].view(m, n // 32)
    P.mxfp8_linear(x, weights, activation=act, residual=res, out=out)
    assert torch.equal(out[0], codes) and torch.equal(out[1], scales)
    assert bool((room[:16] == 93).all()) and bool((room[m * n + 16:] == 93).all())
    assert bool((sroom[:3] == 93).all()) and bool((sroom[m * (n // 32) + 3:] == 93).all())


@pytest.mark.parametrize("m,k,n", [(1, 96, 40), (2, 6144, 1024), (13, 800, 136), (31, 1056, 640), (60, 2048, 264), (64, 512, 4096), (65, 512, 96), (300, 544, 136), (1300, 160, 520)])
def test_bf16_rows_strides_and_in_place(P, m, k, n):
    gen = gen_of(m, k, n)
    wide = torch.randn((m, k + 40), generator=gen, device="cuda").bfloat16()
    x = wide[:, 8:k + 8]
    w = real(gen, n, k, 1.0 / math.sqrt(k))
    weights = P.LinearWeights.from_row_major(*w)
    q = P.mxfp8_quant(x)
    byte = mxfp8_of(x.double(), 1)
    assert torch.equal(q[1].double(), byte)
    assert torch.equal(q[0].view(torch.float8_e4m3fn).float(),
                       (x.double() / torch.exp2(byte - 127).repeat_interleave(32, -1)).float().to(torch.float8_e4m3fn).float())
    plain = P.mxfp8_linear(q, weights)
    assert torch.equal(P.mxfp8_linear(x, weights), plain)
    # infinities and NaN are quantised alike inside the product and in front of it
    odd = x.clone()
    odd[0, 3], odd[m - 1, k - 1], odd[m // 2, 40] = float("inf"), float("-inf"), float("nan")
    got, want = P.mxfp8_linear(odd, weights), P.mxfp8_linear(P.mxfp8_quant(odd), weights)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    # residual rows and result rows inside wider buffers; what is beside them stays as it was
    stream = torch.randn((m + 1, n + 64), generator=gen, device="cuda").bfloat16()
    keep, view = stream.clone(), stream[:m, 16:n + 16]
    res = view.clone()
    want = P.mxfp8_linear(q, weights, residual=res)
    out = torch.full((m + 1, n + 24), 3.0, dtype=torch.bfloat16, device="cuda")
    P.mxfp8_linear(q, weights, residual=view, out=out[:m, 8:n + 8])
    assert torch.equal(out[:m, 8:n + 8], want) and torch.equal(stream, keep)
    assert bool((out[m] == 3).all()) and bool((out[:, :8] == 3).all()) and bool((out[:, n + 8:] == 3).all())
    assert P.mxfp8_linear(q, weights, residual=view, out=view) is view
    keep[:m, 16:n + 16] = want
    assert torch.equal(stream, keep)
    one = x[:1].expand(m, k)
    assert torch.equal(P.mxfp8_linear(one, weights), P.mxfp8_linear(one.contiguous(), weights))


@pytest.mark.parametrize("m,k", [(1, 32), (9, 96), (300, 160), (33, 6144), (5, 8224), (3, 32800), (2, 70016)])
def test_quantised_rows_of_any_width(P, m, k):
    """Exact in 64 bits: the scale's power of two and the code's rounding; rows inside wider rows; scales that begin at any byte."""
    gen = gen_of("quant", m, k)
    x = torch.randn((m, k + 8), generator=gen, device="cuda") * torch.exp(2 * torch.randn((m, k + 8), generator=gen, device="cuda"))
    x = x.bfloat16()[:, :k]
    x[0, :32] = 0
    byte = mxfp8_of(x.double(), 1)
    byte[0, 0] = 1
    want = (x.double() / torch.exp2(byte - 127).repeat_interleave(32, -1)).float().to(torch.float8_e4m3fn).view(torch.uint8)
    room = torch.full((m * (k // 32) + 9,), 93, dtype=torch.uint8, device="cuda")
    scales = room[1:m * (k // 32) + 1].view(m, k // 32)
    codes, s = P.mxfp8_quant(x)
    assert torch.equal(s.double(), byte) and torch.equal(codes & 127, want & 127) and torch.equal(codes, want)
    P.mxfp8_quant(x, out=(codes.zero_(), scales))
    assert torch.equal(scales, s) and torch.equal(codes, want) and int(room[0]) == 93 and bool((room[m * (k // 32) + 1:] == 93).all())


@pytest.mark.parametrize("m,k", [(40, 800), (700, 6144), (130, 160)])
def test_rows_of_a_larger_batch_and_unaligned_scales(P, m, k):
    """A slice of the rows: its scales begin at any byte. Same bits as the rows copied out."""
    gen = gen_of(m, k)
    codes, scales = real(gen, m + 3, k)
    weights = P.LinearWeights.from_row_major(*real(gen, 328, k, 1.0 / math.sqrt(k)))
    assert torch.equal(P.mxfp8_linear((codes[3:], scales[3:]), weights), P.mxfp8_linear((codes[3:].clone(), scales[3:].clone()), weights))
    odd = torch.empty(m * (k // 32) + 1, dtype=torch.uint8, device="cuda")[1:].view(m, k // 32)
    odd.copy_(scales[3:])
    assert torch.equal(P.mxfp8_linear((codes[3:], odd), weights), P.mxfp8_linear((codes[3:].clone(), scales[3:].clone()), weights))


@pytest.mark.parametrize("m", [1, 17, 150, 600, 1400])
def test_rows_and_columns_behind_the_last_stay_as_they_were(P, m):
    gen = gen_of(m)
    x, w = whole(gen, m, 160), whole(gen, 160, 160)
    weights = P.LinearWeights.from_row_major(*w)
    want = P.mxfp8_linear(x, weights, mxfp8_out=True)
    codes = torch.full((m + 200, 160), 93, dtype=torch.uint8, device="cuda")
    scales = torch.full((m + 200, 5), 93, dtype=torch.uint8, device="cuda")
    P.mxfp8_linear(x, weights, out=(codes[:m], scales[:m]))
    assert torch.equal(codes[:m], want[0]) and torch.equal(scales[:m], want[1])
    assert bool((codes[m:] == 93).all()) and bool((scales[m:] == 93).all())
    y = torch.full((m + 200, 160), 3.0, dtype=torch.bfloat16, device="cuda")
    P.mxfp8_linear(x, weights, out=y[:m])
    assert bool((y[m:] == 3).all()) and torch.equal(y[:m], P.mxfp8_linear(x, weights))


@pytest.mark.parametrize("m", [3, 140, 1100])
def test_nan_and_infinite_operands_reach_their_row_only(P, m):
    gen = gen_of(m)
    codes, scales = real(gen, m, 544)
    w = real(gen, 264, 544, 0.05)
    weights = P.LinearWeights.from_row_major(*w)
    clean = P.mxfp8_linear((codes, scales), weights)
    codes[1, 77] = 0x7F   # NaN code
    scales[2, 16] = 255   # NaN scale, in the K-tile that the row fills in part
    got = P.mxfp8_linear((codes, scales), weights)
    assert bool(got[1:3].isnan().all())
    assert torch.equal(got[0], clean[0]) and torch.equal(got[3:], clean[3:])
    wc, ws = w[0].clone(), w[1].clone()
    wc[200, 543] = 0xFF
    got = P.mxfp8_linear((codes, scales), P.LinearWeights.from_row_major(wc, ws))
    assert bool(got[:, 200].isnan().all()) and torch.equal(got[3:, 201:], clean[3:, 201:]) and torch.equal(got[3:, :200], clean[3:, :200])
    x = torch.randn((m, 544), generator=gen, device="cuda").bfloat16()
    x[0, 5] = float("inf")
    c, s = P.mxfp8_quant(x)
    assert int(c[0, 5]) == 0x7E and int(s[0, 0]) == 254 and bool((s[:, 1:] < 130).all())


def test_no_rows(P):
    gen = gen_of(0)
    weights = P.LinearWeights.from_row_major(*real(gen, 64, 96))
    x = torch.empty((0, 96), dtype=torch.uint8, device="cuda"), torch.empty((0, 3), dtype=torch.uint8, device="cuda")
    assert P.mxfp8_linear(x, weights).shape == (0, 64)
    assert P.mxfp8_linear(torch.empty((0, 96), dtype=torch.bfloat16, device="cuda"), weights, mxfp8_out=True)[1].shape == (0, 2)


def test_sums_repeat_and_two_calls_at_once(P):
    """Two streams, the same weights, different rows: nothing is shared between calls; and the same call has the same bits again."""
    gen = gen_of(1)
    weights = P.LinearWeights.from_row_major(*real(gen, 1544, 2048, 0.03))
    xs = [real(gen, m, 2048) for m in (3, 90, 300, 1200)]
    want = [P.mxfp8_linear(x, weights) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[] for _ in xs]
    for _ in range(5):
        for x, st, g in zip(xs, streams, got):
            with torch.cuda.stream(st):
                g.append(P.mxfp8_linear(x, weights))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for g, w in zip(got, want) for y in g)


def test_two_captured_graphs_at_once(P):
    """Graphs of bf16 calls (the rows' codes are the call's own) replayed on two streams, with inputs that change between replays."""
    gen = gen_of(11)
    weights = P.LinearWeights.from_row_major(*real(gen, 1032, 1056, 0.03), torch.randn(1032, generator=gen, device="cuda"))
    ms = (30, 130, 700)
    held = [torch.randn((m, 1056), generator=gen, device="cuda").bfloat16() for m in ms]
    graphs, outs = [], []
    for x in held:
        P.mxfp8_linear(x, weights, activation="silu")
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            outs.append(P.mxfp8_linear(x, weights, activation="silu"))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for x in held:
            x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        torch.cuda.synchronize()
        for _ in range(4):
            for graph, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, P.mxfp8_linear(x, weights, activation="silu")) for x, y in zip(held, outs))


@pytest.mark.parametrize("m", [1, 6, 64, 65, 300, 1100])
def test_columns_of_one_tensor(P, m):
    """Rows, residual and result side by side in one tensor, the result beside and in the residual; what reaches into the rows is refused."""
    gen = gen_of(12, m)
    k, n = 544, 520
    weights = P.LinearWeights.from_row_major(*real(gen, n, k, 0.05))
    buf = torch.randn((m, k + 2 * n), generator=gen, device="cuda").bfloat16()
    x, res, out = buf[:, :k], buf[:, k:k + n], buf[:, k + n:]
    want = P.mxfp8_linear(x.contiguous(), weights, residual=res.contiguous())
    keep = buf.clone()
    assert P.mxfp8_linear(x, weights, residual=res, out=out) is out
    assert torch.equal(out, want) and torch.equal(buf[:, :k + n], keep[:, :k + n])
    P.mxfp8_linear(x, weights, residual=res, out=res)
    assert torch.equal(res, want) and torch.equal(x, keep[:, :k])
    for bad in (buf[:, k - 8:k - 8 + n], buf[:, :n], buf[:, 8:8 + n]):
        with pytest.raises(ValueError):
            P.mxfp8_linear(x, weights, out=bad)
    with pytest.raises(ValueError):
        P.mxfp8_linear(x, weights, residual=res, out=buf[:, k + 8:k + 8 + n])
    torch.cuda.synchronize()
    assert torch.equal(x, keep[:, :k])


@pytest.mark.parametrize("m,stride", [(40, 1 << 26), (300, 1 << 23), (1100, 1 << 21)])
def test_rows_beyond_32_bits(P, m, stride):
    """bf16 rows, residual and result so far apart that the last begin behind 2^31 elements."""
    gen = gen_of(13, m)
    k, n = 544, 264
    weights = P.LinearWeights.from_row_major(*real(gen, n, k, 0.05))
    big = torch.empty((m, stride), dtype=torch.bfloat16, device="cuda")
    x, res = big[:, :k], big[:, 1024:1024 + n]
    x.copy_(torch.randn((m, k), generator=gen, device="cuda"))
    res.copy_(torch.randn((m, n), generator=gen, device="cuda"))
    want = P.mxfp8_linear(x.contiguous(), weights, residual=res.contiguous())
    assert torch.equal(P.mxfp8_linear(x, weights, residual=res), want)
    P.mxfp8_linear(x, weights, residual=res, out=res)
    assert torch.equal(res, want)


def test_codes_beyond_32_bits(P):
    """Codes behind 2^31 bytes in, behind 2^32 bytes out: whole numbers, so that the rows of a smaller call have the same bits."""
    gen = gen_of(14)
    m, k, n = 1100000, 2080, 4096
    x = torch.randint(-2, 3, (m, k), generator=gen, device="cuda", dtype=torch.int8)
    codes = torch.empty((m, k), dtype=torch.uint8, device="cuda")
    for part, to in zip(x.split(100000), codes.split(100000)):
        to.copy_(part.to(torch.bfloat16).to(torch.float8_e4m3fn).view(torch.uint8))
    scales = torch.randint(126, 129, (m, k // 32), generator=gen, device="cuda", dtype=torch.uint8)
    weights = P.LinearWeights.from_row_major(*whole(gen, n, k))
    got = P.mxfp8_linear((codes, scales), weights, activation="relu", mxfp8_out=True)
    for at in (0, 524200, 1048500, m - 300):  # (2^31 / n and 2^32 / n are 524288 and 1048576)
        want = P.mxfp8_linear((codes[at:at + 300], scales[at:at + 300]), weights, activation="relu", mxfp8_out=True)
        assert torch.equal(got[0][at:at + 300], want[0]) and torch.equal(got[1][at:at + 300], want[1])


def test_the_shared_expert_is_two_such_products(P):
    """The same weights through the shared expert: the norm's rows, a gated product to MXFP8, a product to bf16. The first product's
    sums may be ordered differently, so that a code may fall to the other side of a border: the results agree as two roundings do."""
    from amd_kernels_b200.moe.mxfp4_h6144_i768_e128_top4 import shared_expert as S
    gen = gen_of(2)
    w13, w2 = real(gen, 1536, 6144, 0.02), real(gen, 6144, 768, 0.05)
    shared = P.SharedWeights.from_row_major(*w13, *w2)
    l13, l2 = P.LinearWeights.from_row_major(*w13, gated=True), P.LinearWeights.from_row_major(*w2)
    for m in (1, 50, 300, 1700):
        x = torch.randn((m, 6144), generator=gen, device="cuda").bfloat16()
        q = P.mxfp8_quant(x)
        assert all(torch.equal(a, b) for a, b in zip(q, S.shared_quant_rows(x)))
        want = S.shared_expert(x, shared).double()
        got = P.mxfp8_linear(P.mxfp8_linear(q, l13, activation="swiglu_oai", mxfp8_out=True), l2).double()
        # half a step of bf16 on each side where all codes agree; a flipped code (2^-3 of one of 768 terms) moves a sum by a few steps
        assert float((got - want).norm() / want.norm()) < 2.0 ** -8


@pytest.mark.parametrize("m", [1, 40, 500])
def test_a_block_as_a_server_runs_it(P, m):
    """Output projection into the residual stream, norm, dense SwiGLU block, norm, MoE layer, tail, the next projection: eager, and captured
    once and replayed on other inputs, with the same bits; the first half against the formula in 64 bits."""
    gen = gen_of(3, m)
    H, I, A = 6144, 1024, 2048
    from tests.test_gpu_add_rmsnorm import formula as norm_formula
    wo, w13, w2 = real(gen, H, A, 0.02), real(gen, 2 * I, H, 0.02), real(gen, H, I, 0.03)
    lo, l13, l2 = (P.LinearWeights.from_row_major(*w, gated=g) for w, g in ((wo, False), (w13, True), (w2, False)))
    lq = P.LinearWeights.from_row_major(*real(gen, 1280, H, 0.02), torch.randn(1280, generator=gen, device="cuda"))
    weight = (0.1 * torch.randn(H, generator=gen, device="cuda")).bfloat16()
    e = 8
    moe = P.MoeWeights.from_row_major(0.02 * torch.randn((e, H), generator=gen, device="cuda"), None,
                                      *(torch.randint(0, hi, shape, generator=gen, device="cuda", dtype=torch.uint8) + lo_ for shape, lo_, hi in
                                        (((e, 1536, 3072), 0, 256), ((e, 1536, 192), 120, 4), ((e, H, 384), 0, 256), ((e, H, 24), 120, 4))),
                                      routing_mode="softmax")
    P.warm_up_mxfp4_moe(moe)

    def block(attn, stream):
        stream = P.mxfp8_linear(attn, lo, residual=stream)
        first = P.add_rmsnorm_mxfp8(stream, None, weight)
        h = P.mxfp8_linear((first.codes, first.scales), l13, activation="swiglu_oai", mxfp8_out=True)
        down = P.mxfp8_linear(h, l2)
        second = P.add_rmsnorm_mxfp8(down, stream, weight, mxfp8=False, bf16_out=True)
        slots, shared = P.mxfp4_moe(second.normed, moe, return_partials=True)
        tail = P.slots4_add_rmsnorm_mxfp8(slots, shared, second.residual, weight)
        return stream, first, h, down, second, tail, P.mxfp8_linear((tail.codes, tail.scales), lq)

    def inputs():
        return torch.randn((m, A), generator=gen, device="cuda").bfloat16(), torch.randn((m, H), generator=gen, device="cuda").bfloat16()

    attn, stream = inputs()
    got = block(attn, stream)
    q = P.mxfp8_quant(attn)
    y, slack = formula(q, wo, residual=stream)
    assert bool(((got[0].double() - y).abs() <= 2.0 ** -8 * y.abs() + 1.01 * slack).all())
    check_codes(got[1].codes, got[1].scales, norm_formula(got[0], None, weight, 1e-6, 1.0)[1], 0, 2.0 ** -18)
    y, slack = formula((got[1].codes, got[1].scales), w13, act="swiglu_oai")
    check_codes(*got[2], y, 1, 0.0, slack)
    y, slack = formula(got[2], w2)
    assert bool(((got[3].double() - y).abs() <= 2.0 ** -8 * y.abs() + 1.01 * slack).all())
    assert torch.equal(got[4].residual, norm_formula(got[3], got[0], weight, 1e-6, 1.0)[0])
    assert bool(got[6].isfinite().all())
    attn_in, stream_in = attn.clone(), stream.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = block(attn_in, stream_in)
    for _ in range(2):
        attn, stream = inputs()
        attn_in.copy_(attn)
        stream_in.copy_(stream)
        graph.replay()
        torch.cuda.synchronize()
        want = block(attn, stream)
        assert torch.equal(held[0], want[0]) and torch.equal(held[2][0], want[2][0]) and torch.equal(held[5].codes, want[5].codes)
        assert torch.equal(held[6], want[6])
