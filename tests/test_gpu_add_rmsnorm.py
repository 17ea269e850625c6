"""Residual addition, RMS norm and MXFP8 output without slots, against the formula in 64 bits.

The residual out is one rounding of an exact fp32 sum: bit for bit. y: squares are summed in fp32 by threads that add at most 64 of
them one after the other, then at most 5 + 32 partial sums, so the sum is within 101 * 2^-24 of its value relative; half of that
for its root, and at most 8 roundings of 2^-24 behind it: y is within DELTA = 2^-18 (64 * 2^-24) of the formula, relative. bf16(y) adds half a step,
2^-8. A scale byte may differ only where max|y| / 448 is within DELTA of a power of two. A code stands for a value within half a step:
2^-4 relative, 2^-10 of the block's scale below the normal range."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DELTA = 2.0 ** -18


@pytest.fixture(scope="module")
def P():
    from amd_kernels_b200.moe import mxfp4_h6144_i768_e128_top4
    return mxfp4_h6144_i768_e128_top4


def rows(gen, m, h, pad=0, scale=1.0):
    t = torch.empty((m, h + pad), dtype=torch.bfloat16, device="cuda")[:, :h]
    t[:] = torch.randn((m, h), generator=gen, device="cuda") * scale * torch.exp(0.5 * torch.randn(h, generator=gen, device="cuda"))
    return t


def formula(x, residual, weight, eps, offset):
    s = x.float() if residual is None else x.float() + residual.float()
    v = s.double()
    y = v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps) * (weight.double() + offset)
    return s.bfloat16(), y


def mxfp8_of(y, lowest):
    """fp64 -> (E4M3 values in units of the scale, scale bytes)"""
    top = y.unflatten(-1, (-1, 32)).abs().amax(-1).clamp_min(2.0 ** -126)
    byte = torch.ceil(torch.log2(top / 448.0)) + 127
    byte = (byte + (448.0 * torch.exp2(byte - 127) < top) - (448.0 * torch.exp2(byte - 128) >= top).double()).clamp(lowest, 254)
    return byte


def check_codes(codes, scales, y, lowest, delta, slack=0.0):
    """``slack``: an error of y in absolute terms, a tensor like y (or 0)"""
    got_scale = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    low, high = (mxfp8_of(y * (1 + f * delta) + f * slack * torch.sign(y), lowest) for f in (-1, 1))
    top = y.abs() * (1 + delta) + slack
    high = mxfp8_of(top, lowest)
    low = mxfp8_of((y.abs() * (1 - delta) - slack).clamp_min(0), lowest)
    assert bool(((scales >= low) & (scales <= high)).all())
    v = codes.view(torch.float8_e4m3fn).double() * got_scale
    assert bool(((v - y).abs() <= (2.0 ** -4 + 2 * delta) * y.abs() + 2.0 ** -10 * got_scale + 2 * slack).all())


WIDTHS = [32, 64, 96, 256, 288, 544, 1024, 1056, 2080, 4064, 4096, 6144, 6176, 8192, 16384, 16416, 32768]


@pytest.mark.parametrize("h", WIDTHS)
@pytest.mark.parametrize("m", [1, 2, 9, 67])
def test_against_the_formula(P, m, h):
    gen = torch.Generator(device="cuda").manual_seed(m * 100003 + h)
    x, res = rows(gen, m, h), rows(gen, m, h, scale=3.0)
    weight = (0.2 * torch.randn(h, generator=gen, device="cuda")).bfloat16()
    got = P.add_rmsnorm_mxfp8(x, res, weight, 1e-5, bf16_out=True)
    want_res, y = formula(x, res, weight, 1e-5, 1.0)
    assert torch.equal(got.residual, want_res)
    assert bool(((got.normed.double() - y).abs() <= (2.0 ** -8 + 2 * DELTA) * y.abs()).all())
    check_codes(got.codes, got.scales, y, 0, DELTA)


@pytest.mark.parametrize("m,h,pad", [(5, 6144, 8), (130, 4064, 544), (3, 96, 32)])
@pytest.mark.parametrize("offset", [0.0, 1.0])
@pytest.mark.parametrize("with_residual", [False, True])
def test_strides_offsets_and_outputs(P, m, h, pad, offset, with_residual):
    gen = torch.Generator(device="cuda").manual_seed(h + pad)
    x = rows(gen, m, h, pad)
    res = rows(gen, m, h, 3 * pad) if with_residual else None
    weight = (1.0 - offset + 0.1 * torch.randn(h, generator=gen, device="cuda")).bfloat16()
    want_res, y = formula(x, res, weight, 1e-6, offset)
    full = P.add_rmsnorm_mxfp8(x, res, weight, weight_offset=offset, bf16_out=True)
    assert (full.residual is None) == (res is None) and (res is None or torch.equal(full.residual, want_res))
    assert bool(((full.normed.double() - y).abs() <= (2.0 ** -8 + 2 * DELTA) * y.abs()).all())
    only8 = P.add_rmsnorm_mxfp8(x, res, weight, weight_offset=offset)
    only16 = P.add_rmsnorm_mxfp8(x, res, weight, weight_offset=offset, mxfp8=False, bf16_out=True)
    assert only8.normed is None and torch.equal(only8.codes, full.codes) and torch.equal(only8.scales, full.scales)
    assert only16.codes is None and only16.scales is None and torch.equal(only16.normed, full.normed)
    # results in rows of wider buffers, whose other columns stay as they were
    big = torch.full((m + 2, h + 40), 7.0, dtype=torch.bfloat16, device="cuda")
    keep = big.clone()
    view = big[1:m + 1, 8:h + 8]
    P.add_rmsnorm_mxfp8(x, res, weight, weight_offset=offset, out=P.TailOutput(None, None, None, view))
    assert torch.equal(view, full.normed)
    keep[1:m + 1, 8:h + 8] = full.normed
    assert torch.equal(big, keep)


def test_in_place_and_shared_residual(P):
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, res = rows(gen, 33, 6144), rows(gen, 33, 6144)
    weight = (0.1 * torch.randn(6144, generator=gen, device="cuda")).bfloat16()
    want = P.add_rmsnorm_mxfp8(x, res, weight, bf16_out=True)
    stream, normed = res.clone(), x.clone()
    out = P.TailOutput(stream, torch.empty_like(want.codes), torch.empty_like(want.scales), normed)
    assert P.add_rmsnorm_mxfp8(normed, stream, weight, out=out) is out
    assert all(torch.equal(a, b) for a, b in zip((out.residual, out.codes, out.scales, out.normed),
                                                 (want.residual, want.codes, want.scales, want.normed)))
    one = res[:1].expand(33, 6144)
    assert torch.equal(P.add_rmsnorm_mxfp8(x, one, weight).codes, P.add_rmsnorm_mxfp8(x, one.contiguous(), weight).codes)


def test_columns_of_one_tensor(P):
    """Input and results side by side in one tensor; a result that reaches into an input is refused."""
    gen = torch.Generator(device="cuda").manual_seed(15)
    m, h = 37, 1056
    weight = (0.1 * torch.randn(h, generator=gen, device="cuda")).bfloat16()
    buf = rows(gen, m, 4 * h)
    x, res, res_out, normed = buf.split(h, 1)
    want = P.add_rmsnorm_mxfp8(x.contiguous(), res.contiguous(), weight, mxfp8=False, bf16_out=True)
    keep = buf.clone()
    P.add_rmsnorm_mxfp8(x, res, weight, out=P.TailOutput(res_out, None, None, normed))
    assert torch.equal(res_out, want.residual) and torch.equal(normed, want.normed) and torch.equal(buf[:, :2 * h], keep[:, :2 * h])
    for bad in (buf[:, h - 8:2 * h - 8], buf[:, 8:h + 8], buf[:, 2 * h - 8:3 * h - 8]):
        with pytest.raises(ValueError):
            P.add_rmsnorm_mxfp8(x, res, weight, out=P.TailOutput(None, None, None, bad))
    with pytest.raises(ValueError):
        P.add_rmsnorm_mxfp8(x, res, weight, out=P.TailOutput(res_out, None, None, buf[:, 2 * h + 8:3 * h + 8]))


def test_bits_of_the_tail_and_of_a_row_alone(P):
    """With one slot that is not zero the tail's sum is that slot, and its other steps are these; a row alone has the bits it has among others."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    x, res = rows(gen, 70, 6144), rows(gen, 70, 6144)
    weight = (0.1 * torch.randn(6144, generator=gen, device="cuda")).bfloat16()
    slots = torch.zeros((70, 4, 6144), dtype=torch.bfloat16, device="cuda")
    slots[:, 2] = x
    want = P.slots4_add_rmsnorm_mxfp8(slots, None, res, weight, 1e-6, bf16_out=True)
    got = P.add_rmsnorm_mxfp8(x, res, weight, 1e-6, bf16_out=True)
    for key in ("residual", "codes", "scales", "normed"):
        assert torch.equal(getattr(got, key), getattr(want, key)), key
    alone = P.add_rmsnorm_mxfp8(x[41:42], res[41:42], weight, 1e-6)
    assert torch.equal(alone.codes[0], got.codes[41]) and torch.equal(alone.scales[0], got.scales[41])


def test_zero_rows_infinities_and_nan(P):
    x = torch.randn((5, 512), device="cuda").bfloat16()
    x[0] = 0.0
    x[1, 7] = float("inf")
    x[2, 300] = float("nan")
    x[3] = 1e-30
    res, weight = torch.zeros_like(x), torch.zeros(512, dtype=torch.bfloat16, device="cuda")
    got = P.add_rmsnorm_mxfp8(x, res, weight, 1e-6, bf16_out=True)
    assert bool((got.normed[0] == 0).all()) and bool((got.codes[0] & 127 == 0).all()) and bool((got.scales[0] < 127).all())
    assert bool(got.normed[1, 7].isnan()) and bool((got.normed[1, :7] == 0).all())  # 1 / sqrt(inf) is 0, and inf * 0 is NaN
    assert bool(got.normed[2].isnan().all()) and bool((got.codes[2] & 127 == 127).all())
    assert bool(((got.normed[3].double() - x[3].double() * 1e3).abs() <= 2.0 ** -7 * 1e-27).all())  # eps keeps tiny rows tiny
    y4 = formula(x[4:], res[4:], weight, 1e-6, 1.0)[1]
    assert bool(((got.normed[4:].double() - y4).abs() <= (2.0 ** -8 + 2 * DELTA) * y4.abs()).all())


def test_no_rows_and_rows_behind_the_last(P):
    weight = torch.zeros(64, dtype=torch.bfloat16, device="cuda")
    none = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")
    got = P.add_rmsnorm_mxfp8(none, none, weight, bf16_out=True)
    assert got.residual.shape == (0, 64) and got.codes.shape == (0, 64) and got.scales.shape == (0, 2) and got.normed.shape == (0, 64)
    # eight rows share a CTA at this width: the rows behind the ninth stay as they were
    x = torch.randn((9, 64), device="cuda").bfloat16()
    codes = torch.full((16, 64), 93, dtype=torch.uint8, device="cuda")
    scales = torch.full((16, 2), 93, dtype=torch.uint8, device="cuda")
    P.add_rmsnorm_mxfp8(x, None, weight, out=P.TailOutput(None, codes[:9], scales[:9], None))
    assert bool((codes[9:] == 93).all()) and bool((scales[9:] == 93).all()) and not bool((codes[:9] == 93).all())


def test_offsets_beyond_32_bits(P):
    """Rows 2^17 elements apart: the last ones begin behind 2^32 elements."""
    m, h = 33000, 64
    big = torch.zeros((m, 1 << 17), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn((m, h), generator=gen, device="cuda").bfloat16()
    big[:, :h] = x
    weight = torch.zeros(h, dtype=torch.bfloat16, device="cuda")
    got, want = P.add_rmsnorm_mxfp8(big[:, :h], None, weight), P.add_rmsnorm_mxfp8(x, None, weight)
    assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)


def test_graph_and_other_stream(P):
    gen = torch.Generator(device="cuda").manual_seed(9)
    x, res = rows(gen, 40, 6144), rows(gen, 40, 6144)
    weight = (0.1 * torch.randn(6144, generator=gen, device="cuda")).bfloat16()
    want = P.add_rmsnorm_mxfp8(x, res, weight)
    x_in = x.clone()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = P.add_rmsnorm_mxfp8(x, res, weight)
        with torch.cuda.graph(graph, stream=side):
            got = P.add_rmsnorm_mxfp8(x_in, res, weight)
    side.synchronize()
    assert torch.equal(other.codes, want.codes)
    for _ in range(2):
        got.codes.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got.codes, want.codes) and torch.equal(got.residual, want.residual)
    x_in.copy_(res)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got.codes, P.add_rmsnorm_mxfp8(res, res, weight).codes)
