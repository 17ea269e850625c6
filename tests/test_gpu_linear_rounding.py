"""The arithmetic of the MXFP8 product's activations, seen closer than one result of 8 bits shows it.

Rows of zeros make every sum the bias, exactly; a residual of minus the bf16 value next to the activation leaves their difference, which
is exact in fp32 (both lie within a factor of two). Columns are taken where the activation lies within 2^-17 (relative) of a bf16 value: the
result's own half step, 2^-8 of the difference, is then below 2^-24 of the activation.

u = 2^-24, half a step of fp32. An approximate exponential is within 2^-22 (4 u), a reciprocal within one unit in the last place (2 u).
  p sigmoid(v), exponent w = -v log2(e) off by A u relative (constants, products; A = 2 for v = c p, 8 for the cubic of the tanh form):
      (1 - sigmoid) (ln 2 |w| A + 4) u from the exponential, then sum u, reciprocal 2 u, product u, and 2 u where a gate meets its up.
  p Phi(p) = max(p, 0) - |p| e, e = erfc(z) / 2 = exp(-z^2) t Q(t) / 2 off by: the fit's 6.7e-8 (1.2 u); t 4 u, times the slope
      d ln(t Q) / d ln t <= 2.7; a polynomial of degree 7 at most 14.6 u (the sum of (2 i + 1) |c_i| t^i over Q, largest at t = 1); the
      exponent x = z^2 log2(e) + 1 three roundings, 3 ln 2 x u; the exponential 4 u; two products 2 u: (33 + 3 ln 2 x) u of |p| e; and u of the sum."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def P():
    from amd_kernels_b200.moe import mxfp4_h6144_i768_e128_top4
    return mxfp4_h6144_i768_e128_top4


def formula(p, act):
    """(the activation, the bound on its error) in 64 bits; gated ones with an up of 1 (SwiGLU) or 0 (the clamped form)"""
    if act == "gelu":
        e = torch.special.erfc(p.abs() * math.sqrt(0.5)) / 2
        y = p.clamp_min(0) - p.abs() * e
        return y, (33 + 3 * math.log(2) * (p * p * 0.5 / math.log(2) + 1)) * U * p.abs() * e + U * y.abs()
    v, roundings = {"gelu_tanh": (2 * math.sqrt(2 / math.pi) * (p + 0.044715 * p ** 3), 8), "swiglu_oai": (1.702 * p, 3)}.get(act, (p, 2))
    s = torch.sigmoid(v)
    y = p * s
    return y, ((1 - s) * (v.abs() * roundings + 4) + 6) * U * y.abs()


@pytest.mark.parametrize("act", ["gelu", "silu", "gelu_tanh", "swiglu", "swiglu_oai"])
@pytest.mark.parametrize("m", [1, 100, 300])
def test_activations_to_32_bits(P, m, act):
    gen = torch.Generator(device="cuda").manual_seed(17)
    p = torch.rand(1 << 22, generator=gen, device="cuda") * 9.0 - 3.5
    y, _ = formula(p.double(), act)
    near = y.float().bfloat16().double()
    p = p[(y - near).abs() <= 2.0 ** -17 * y.abs()]
    n = min(p.numel() // 64 * 64, 8192)
    p = p[:n]
    assert n >= 4096
    y, bound = formula(p.double(), act)
    near = y.float().bfloat16()
    gated = act.startswith("swiglu")
    bias = torch.cat([p, torch.full_like(p, float(act == "swiglu"))]) if gated else p
    w = P.LinearWeights.from_row_major(torch.zeros((bias.numel(), 32), dtype=torch.uint8, device="cuda"),
                                       torch.full((bias.numel(), 1), 127, dtype=torch.uint8, device="cuda"), bias, gated=gated)
    x = torch.zeros((m, 32), dtype=torch.uint8, device="cuda"), torch.full((m, 1), 127, dtype=torch.uint8, device="cuda")
    got = P.mxfp8_linear(x, w, activation=act, residual=(-near).expand(m, n).contiguous()).double()
    error = (got + near.double() - y).abs()
    slack = 2.0 ** -8 * ((y - near.double()).abs() + bound)
    assert bool((error <= bound + slack).all()), float((error / bound).max())
