"""The MXFP8 product of up to 128 rows by more weight tiles than run at once (a projection as wide as a vocabulary): the one-CTA kernel without
a split of K, in several rounds, where a CTA takes over the shared and tensor memory of one that has left. Whole numbers: bit for bit."""
import pytest
import torch

from tests.test_gpu_add_rmsnorm import mxfp8_of
from tests.test_gpu_linear import P, gen_of, no_wait_ran_out, values, whole  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def inputs(m, k, n):
    gen = gen_of("rounds", m, k, n)
    bias = torch.randint(-8, 9, (n,), generator=gen, device="cuda").float()
    return gen, whole(gen, m, k), whole(gen, n, k), bias


@pytest.mark.parametrize("m,k,n", [(1, 96, 50008), (16, 1056, 38016), (33, 160, 50016), (64, 544, 76000), (65, 96, 40008), (128, 288, 50016)])
def test_several_rounds_bit_for_bit(P, m, k, n):  # noqa: F811
    gen, x, w, bias = inputs(m, k, n)
    res = torch.randint(-64, 65, (m, n), generator=gen, device="cuda").bfloat16()
    weights = P.LinearWeights.from_row_major(*w, bias)
    p = values(*x) @ values(*w).t() + bias.double()
    for _ in range(3):  # launch behind launch
        y, with_residual = P.mxfp8_linear(x, weights), P.mxfp8_linear(x, weights, activation="relu", residual=res)
    assert torch.equal(y, p.float().bfloat16())
    assert torch.equal(with_residual, (p.clamp_min(0) + res.double()).float().bfloat16())
    if n % 32 == 0:
        codes, scales = P.mxfp8_linear(x, weights, mxfp8_out=True)
        byte = mxfp8_of(p, 1)
        assert torch.equal(scales.double(), byte)
        want = (p / torch.exp2(byte - 127).repeat_interleave(32, -1)).float().to(torch.float8_e4m3fn)
        assert torch.equal(codes.view(torch.float8_e4m3fn).float(), want.float())


@pytest.mark.parametrize("m,k,n", [(1, 96, 50008), (16, 1056, 40000), (40, 160, 50016), (64, 288, 76000)])
def test_rows_quantised_inside_in_several_rounds(P, m, k, n):  # noqa: F811
    """bf16 rows of whole numbers below 8 are their own MXFP8 values (three bits of mantissa); some rows all zero."""
    gen, _, w, bias = inputs(m, k, n)
    x = torch.randint(-7, 8, (m, k), generator=gen, device="cuda").bfloat16()
    x[::5] = 0
    weights = P.LinearWeights.from_row_major(*w, bias)
    p = x.double() @ values(*w).t() + bias.double()
    for _ in range(3):
        y = P.mxfp8_linear(x, weights)
    assert torch.equal(y, p.float().bfloat16())


def test_rounds_behind_and_in_front_of_other_calls(P):  # noqa: F811
    """Norm, wide gated product, product back, each reading what the one before wrote, without a wait between them; then with one. The same in a
    captured graph."""
    gen, _, w, bias = inputs(48, 1024, 81920)
    down = P.LinearWeights.from_row_major(*whole(gen, 1024, 40960))
    wide = P.LinearWeights.from_row_major(*w, bias, gated=True)
    x = torch.randn((48, 1024), generator=gen, device="cuda").bfloat16()
    weight = torch.zeros(1024, dtype=torch.bfloat16, device="cuda")

    def block(wait):
        got = []
        for _ in range(3):
            normed = P.add_rmsnorm_mxfp8(x, None, weight)
            wait()
            h = P.mxfp8_linear((normed.codes, normed.scales), wide, activation="swiglu", mxfp8_out=True)
            wait()
            got += [*h, P.mxfp8_linear(h, down, residual=x)]
            wait()
        return got

    want = block(torch.cuda.synchronize)
    for got in (block(lambda: None), block(lambda: None)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = block(lambda: None)
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
