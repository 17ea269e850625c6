"""Refusals of the norm without slots and of the MXFP8 product, without a GPU: the entry points' own checks and the C ABI's."""
import ctypes

import pytest
import torch

from amd_kernels_b200 import _lib
from amd_kernels_b200.moe import mxfp4_h6144_i768_e128_top4 as P
from amd_kernels_b200.moe import mxfp4_h6144_i1536_e128_top4 as P2
from amd_kernels_b200.moe.mxfp4_h6144_i768_e128_top4 import linear as L

BF16, U8 = torch.bfloat16, torch.uint8


def at(a):
    return None if a is None else ctypes.c_void_p(a)


def test_both_packages_have_them():
    for name in ("TailOutput", "add_rmsnorm_mxfp8", "LinearWeights", "mxfp8_linear", "mxfp8_quant"):
        assert name in P.__all__ and name in P2.__all__ and getattr(P, name) is getattr(P2, name)


def refused(call, *args, why=None, **kw):
    """A ValueError; for another reason than that nothing is launched on host tensors, unless ``why`` says so."""
    with pytest.raises(ValueError) as e:
        call(*args, **kw)
    assert ("nothing is launched" in str(e.value)) == (why == "nothing is launched"), str(e.value)


# ------------------------------------------------------------------------------------------------ the norm
def norm_call(lib, x=4096, xs=64, r=1 << 20, rs=64, w=256, rows=4, h=64, ro=2 << 20, ros=64, n=3 << 20, ns=64, c=4 << 20, s=5 << 20):
    p = [0 if a is None else a for a in (x, r, w, ro, n, c, s)]
    return lib.b200moe_add_rmsnorm_quant(_lib.NORM_CALL.pack(p[0], xs, p[1], rs, p[2], p[3], ros, p[4], ns, p[5], p[6], rows, h, 1.0, 1e-6), None)


@pytest.mark.parametrize("inter", [768, 1536])
def test_c_abi_refuses_norm_arguments(inter):
    lib = _lib.load(inter)
    A, L_ = _lib.E_ARG, _lib.E_ALIGN
    for bad in (dict(x=None), dict(w=None), dict(rows=-1), dict(h=0), dict(h=48), dict(h=32800), dict(c=None), dict(s=None),
                dict(r=None), dict(ro=None, n=None, c=None, s=None), dict(xs=56), dict(rs=56), dict(ros=0), dict(ns=32), dict(xs=0)):
        assert norm_call(lib, **bad) == A, bad
    for bad in (dict(x=4104), dict(r=(1 << 20) + 2), dict(w=264), dict(ro=(2 << 20) + 8), dict(n=(3 << 20) + 8), dict(c=(4 << 20) + 4),
                dict(xs=68), dict(rs=65), dict(ros=66), dict(ns=70)):
        assert norm_call(lib, **bad) == L_, bad
    # overlaps: only the very rows of x or residual may be written
    for bad in (dict(ro=4096 + 128), dict(n=(1 << 20) + 128), dict(n=2 << 20), dict(c=4096), dict(s=(4 << 20) + 8), dict(ro=4096, ros=72),
                dict(r=1 << 20, rs=0, ro=1 << 20), dict(n=256 - 128), dict(c=(2 << 20) + 400)):
        assert norm_call(lib, **bad) == A, bad
    assert norm_call(lib, rows=0, x=None, r=None, w=None, ro=None, n=None, c=None, s=None) == 0


def norm_inputs(m=4, h=64):
    return torch.zeros((m, h), dtype=BF16), torch.zeros((m, h), dtype=BF16), torch.zeros(h, dtype=BF16)


def test_norm_refuses_bad_tensors():
    x, r, w = norm_inputs()
    out = lambda **k: P.TailOutput(**{"residual": None, "codes": None, "scales": None, "normed": None, **k})  # noqa: E731
    for args, kw in [((x.float(), r, w), {}), ((x[0], r, w), {}), ((x, r[:3], w), {}), ((x, r.float(), w), {}), ((x, r, w[:32]), {}),
                     ((x, r, w.float()), {}), ((x, r, w[None]), {}), ((x[:, :48], r[:, :48], w[:48]), {}),
                     ((x[:, ::2], r[:, ::2], w[:32]), {}), ((x[:1].expand(4, 64), r, w), {}),
                     ((torch.zeros((4, 68), dtype=BF16)[:, :64], r, w), {}), ((x, r, w), dict(out=out())),
                     ((x, None, w), dict(mxfp8=False)), ((x, None, w), dict(out=out(residual=torch.zeros_like(x)))),
                     ((x, r, w), dict(out=out(codes=torch.zeros((4, 64), dtype=U8)))),
                     ((x, r, w), dict(out=out(codes=torch.zeros((4, 64), dtype=U8), scales=torch.zeros((4, 3), dtype=U8)))),
                     ((x, r, w), dict(out=out(codes=torch.zeros((4, 64), dtype=torch.int16), scales=torch.zeros((4, 2), dtype=U8)))),
                     ((x, r, w), dict(out=out(normed=torch.zeros((4, 64))))),
                     ((x, r[::2], w), {}), ((x, r, torch.zeros(128, dtype=BF16)[::2]), {})]:
        refused(P.add_rmsnorm_mxfp8, *args, **kw)
    refused(P.add_rmsnorm_mxfp8, x, r, w, why="nothing is launched")  # all is well but that the tensors are the host's
    refused(P.add_rmsnorm_mxfp8, x, None, w, out=out(normed=x), why="nothing is launched")


# ------------------------------------------------------------------------------------------------ the product
def weights(rows=64, k=96, gated=False, bias=False):
    tiles = torch.zeros((1, 1, 16896), dtype=U8)
    return P.LinearWeights(tiles, torch.zeros(rows) if bias else None, rows, k, gated)


def linear_call(lib, rows=64, k=96, gated=0, tiles=256, bias=None, c=1 << 20, s=2 << 20, m=4, act=0, r=None, rs=64, o=3 << 20, os=64,
                oc=None, osc=None, status=256, x=None, xs=96):
    p = [0 if a is None else a for a in (tiles, bias, c, s, r, o, oc, osc)]
    return lib.b200moe_linear(_lib.LINEAR_CALL.pack(p[0], p[1], rows, k, gated, 0 if x is None else x, xs, p[2], p[3], m, p[4], rs, p[5], os,
                                                    p[6], p[7], act), at(status), None)


@pytest.mark.parametrize("inter", [768, 1536])
def test_c_abi_refuses_product_arguments(inter):
    lib = _lib.load(inter)
    A, L_ = _lib.E_ARG, _lib.E_ALIGN
    for bad in (dict(c=None), dict(s=None), dict(o=None), dict(status=None), dict(tiles=None), dict(m=-1), dict(m=(1 << 24) + 1), dict(k=0),
                dict(k=40), dict(k=(1 << 20) + 32), dict(rows=0), dict(rows=60), dict(rows=(1 << 20) + 8), dict(act=7), dict(act=-1), dict(act=5),
                dict(gated=1), dict(gated=1, act=3), dict(rows=32, gated=1, act=5), dict(oc=4 << 20), dict(o=None, oc=4 << 20),
                dict(oc=4 << 20, osc=5 << 20), dict(rows=40, o=None, oc=4 << 20, osc=5 << 20), dict(os=56), dict(r=4 << 20, rs=8), dict(r=4 << 20, rs=0),
                dict(rows=1 << 20, k=1 << 20)):
        assert linear_call(lib, **bad) == A, bad
    for bad in (dict(tiles=272), dict(c=(1 << 20) + 8), dict(o=(3 << 20) + 8), dict(os=68), dict(r=(4 << 20) + 8), dict(r=4 << 20, rs=66),
                dict(o=None, oc=(4 << 20) + 8, osc=5 << 20), dict(bias=264)):
        assert linear_call(lib, **bad) == L_, bad
    # overlaps: out may be the residual's rows and nothing else that is read
    for bad in (dict(o=1 << 20), dict(o=(2 << 20) - 16), dict(r=3 << 20, rs=72), dict(r=(3 << 20) + 128), dict(r=3 << 20, rs=0),
                dict(o=None, oc=1 << 20, osc=5 << 20), dict(o=None, oc=4 << 20, osc=(4 << 20) + 100), dict(o=None, oc=4 << 20, osc=2 << 20),
                dict(o=None, oc=4 << 20, osc=5 << 20, r=4 << 20)):
        assert linear_call(lib, **bad) == A, bad
    assert linear_call(lib, x=(6 << 20) + 8) == L_ and linear_call(lib, x=6 << 20, xs=100) == L_ and linear_call(lib, x=6 << 20, xs=88) == A
    # bf16 rows: up to 64 need no room for their codes, and then may not be the result's
    assert linear_call(lib, m=65, x=6 << 20, c=None) == A and linear_call(lib, x=6 << 20, o=(6 << 20) + 128, c=None, s=None) == A
    assert linear_call(lib, x=6 << 20, c=None, s=None, status=None) == A
    assert linear_call(lib, m=0, c=None, s=None, o=None) == 0
    for rows, k, gated, want in ((64, 96, 0, 16896), (136, 160, 0, 4 * 16896), (64, 32, 1, 16896), (192, 128, 1, 2 * 16896), (64, 40, 0, 0),
                                 (60, 96, 0, 0), (96, 96, 1, 0), (1 << 20, 1 << 20, 0, 0)):
        assert lib.b200moe_linear_weight_bytes(rows, k, gated) == want
    assert lib.b200moe_preshuffle_linear(at(256), at(256), 64, 96, 0, None, None) == A
    assert lib.b200moe_preshuffle_linear(at(256), at(256), 60, 96, 0, at(256), None) == A
    assert lib.b200moe_preshuffle_linear(at(264), at(256), 64, 96, 0, at(256), None) == L_
    assert lib.b200moe_preshuffle_linear(at(256), at(256), 64, 96, 0, at(272), None) == L_
    quant = lambda x=256, st=96, m=4, k=96, c=4096, s=8192: lib.b200moe_quant_mxfp8(at(x), st, m, k, at(c), at(s), None)  # noqa: E731
    assert all(quant(**bad) == A for bad in (dict(x=None), dict(c=None), dict(s=None), dict(m=-1), dict(k=40), dict(k=0), dict(st=88)))
    assert all(quant(**bad) == L_ for bad in (dict(x=264), dict(st=100), dict(c=4100)))
    assert quant(m=0, x=None) == 0


def test_product_refuses_bad_tensors():
    u8 = lambda *s: torch.zeros(s, dtype=U8)  # noqa: E731
    bf = lambda *s: torch.zeros(s, dtype=BF16)  # noqa: E731
    x = u8(4, 96), u8(4, 3)
    w, g = weights(), weights(gated=True)
    for args, kw in [((x, w), dict(activation="tanh")), ((x, w), dict(activation="swiglu")), ((x, g), {}), ((x, g), dict(activation="relu")),
                     (((u8(4, 64), u8(4, 2)), w), {}), (((u8(4, 96), u8(4, 4)), w), {}), (((u8(4, 96), u8(3, 3)), w), {}),
                     (((u8(4, 192)[:, ::2], u8(4, 3)), w), {}), (((bf(4, 96), u8(4, 3)), w), {}), (((u8(4, 96), None), w), {}),
                     ((bf(4, 64), w), {}), ((bf(96), w), {}), ((torch.zeros((4, 96)), w), {}), (("x", w), {}),
                     ((x, w), dict(residual=bf(4, 32))), ((x, w), dict(residual=bf(3, 64))), ((x, w), dict(residual=torch.zeros((4, 64)))),
                     ((x, w), dict(residual=bf(4, 68)[:, :64])), ((x, w), dict(residual=bf(1, 64).expand(4, 64))), ((x, w), dict(out=bf(4, 72))), ((x, w), dict(out=torch.zeros((4, 64)))),
                     ((x, w), dict(out=bf(1, 64).expand(4, 64))), ((x, w), dict(out=(u8(4, 64), u8(4, 3)))), ((x, w), dict(out=(u8(4, 64), None))),
                     ((x, w), dict(out=(None, None))), ((x, weights(rows=40)), dict(mxfp8_out=True)),
                     ((x, g), dict(activation="swiglu", residual=bf(4, 64))), ((bf(4, 100)[:, :96], w), {})]:
        refused(P.mxfp8_linear, *args, **kw)
    for bad in (bf(4, 40), bf(96), u8(4, 96), torch.zeros((4, 96)), bf(4, 200)[:, ::2], bf(4, 100)[:, :96]):
        refused(P.mxfp8_quant, bad)
    for args, kw in [((x, w), {}), ((bf(4, 96), w), dict(residual=bf(4, 64))), ((x, g), dict(activation="swiglu_oai", mxfp8_out=True))]:
        refused(P.mxfp8_linear, *args, **kw, why="nothing is launched")
    refused(P.mxfp8_quant, bf(4, 96), why="nothing is launched")


def test_weights_refuse_bad_tensors():
    u8 = lambda *s: torch.zeros(s, dtype=U8)  # noqa: E731
    for args in ((u8(64, 96), u8(64, 3)), (torch.zeros(64, 96), u8(64, 3)), (u8(64), u8(64, 3))):
        with pytest.raises(ValueError):
            P.LinearWeights.from_row_major(*args)  # host tensors, types, ranks


def test_output_columns():
    assert weights(gated=True).n == 32 and weights().n == 64 and L.MAX_DIM == 1 << 20


@pytest.mark.parametrize("inter", [768, 1536])
def test_c_abi_refuses_overlaps_with_all_that_is_read(inter):
    """bf16 rows at every size (whether a launch in front quantises them or not), weights and bias; and rows of one stride side by side
    that reach into one another."""
    lib = _lib.load(inter)
    X = 6 << 20
    for m in (4, 64, 65, 300):
        for bad in (dict(o=X), dict(o=X + 96 * 2 * m - 16), dict(xs=160, os=160, o=X + 2 * 88), dict(xs=160, os=160, o=X - 2 * 56), dict(xs=0, o=X)):
            assert linear_call(lib, m=m, x=X, c=8 << 20, s=9 << 20, **bad) == _lib.E_ARG, (m, bad)
    assert linear_call(lib, o=256 + 16512) == _lib.E_ARG and linear_call(lib, bias=3 << 20) == _lib.E_ARG
    assert linear_call(lib, o=3 << 20, os=128, r=(3 << 20) + 112, rs=128) == _lib.E_ARG
    assert linear_call(lib, o=(3 << 20) + 144, os=128, r=3 << 20, rs=128) == _lib.E_ARG  # its end reaches the next row's begin
    quant = lambda x, st, c, s: lib.b200moe_quant_mxfp8(at(x), st, 4, 96, at(c), at(s), None)  # noqa: E731
    assert quant(X, 96, X + 96 * 8 - 8, 8 << 20) == _lib.E_ARG and quant(X, 96, 8 << 20, X + 5) == _lib.E_ARG and quant(X, 96, 8 << 20, (8 << 20) + 300) == _lib.E_ARG
    assert quant(X, 0, X + 96, 8 << 20) == _lib.E_ARG


@pytest.mark.parametrize("inter", [768, 1536])
def test_c_abi_refuses_a_scratch_over_what_the_product_reads(inter):
    """More than 64 bf16 rows are quantised into codes8 and scales8 in front of the product: neither may reach into what it reads then."""
    lib = _lib.load(inter)
    X, C, S, R, W, B = 6 << 20, 8 << 20, 9 << 20, 10 << 20, 11 << 20, 12 << 20
    for m in (65, 300):
        for over, end in ((R, 2 * 64 * m), (W, 16896), (B, 4 * 64), (X, 2 * 96 * m)):
            for bad in (dict(c=over), dict(s=over), dict(c=over + end - 16), dict(s=over + end - 1), dict(c=over - 96 * m + 16), dict(s=over - 3 * m + 1)):
                call = dict(m=m, x=X, c=C, s=S, r=R, tiles=W, bias=B)
                call.update(bad)
                assert linear_call(lib, **call) == _lib.E_ARG, (m, bad)
        assert linear_call(lib, m=m, x=X, c=C, s=C + 96 * m - 1, r=R, tiles=W, bias=B) == _lib.E_ARG
    # a residual of rows that are wider apart: the scratch may not lie in its gaps either (their strides differ)
    assert linear_call(lib, m=300, x=X, c=R + 160, s=S, r=R, rs=512, tiles=W, bias=B) == _lib.E_ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="stands for a device on which no CTA pair can be resident")
@pytest.mark.parametrize("inter", [768, 1536])
def test_without_resident_pairs_the_one_cta_kernel_takes_many_rows(inter):
    """The one-CTA kernel takes any size. Here its launch fails for want of a device; the pair kernel would have said E_DRIVER."""
    lib = _lib.load(inter)
    for call in (dict(m=300, c=8 << 20, s=9 << 20), dict(m=300, c=8 << 20, s=9 << 20, act=3), dict(m=300, c=8 << 20, s=9 << 20, gated=1, act=5),
                 dict(m=5000, c=8 << 20, s=9 << 20, o=None, oc=16 << 20, osc=12 << 20)):
        one_row = linear_call(lib, **{**call, "m": 1})
        assert one_row > 0 and linear_call(lib, **call) == one_row  # a CUDA error code, the same for one row


OTHER_BYTES = [torch.int8, torch.bool, torch.float8_e5m2, torch.float8_e4m3fnuz, torch.float8_e5m2fnuz]


@pytest.mark.parametrize("dtype", OTHER_BYTES + [torch.float8_e8m0fnu])
def test_codes_of_another_format_are_refused(dtype):
    """The same byte stands for another value in the other formats (E4M3FNUZ: half of it)."""
    u8 = lambda *s: torch.zeros(s, dtype=U8)  # noqa: E731
    w, bad = weights(), u8(4, 96).view(dtype)
    refused(P.mxfp8_linear, (bad, u8(4, 3)), w)
    refused(P.mxfp8_linear, (u8(4, 96), u8(4, 3)), w, out=(u8(4, 64).view(dtype), u8(4, 2)))
    refused(P.mxfp8_quant, torch.zeros((4, 96), dtype=BF16), out=(bad, u8(4, 3)))
    x, r, nw = norm_inputs()
    refused(P.add_rmsnorm_mxfp8, x, r, nw, out=P.TailOutput(None, u8(4, 64).view(dtype), u8(4, 2), None))
    with pytest.raises(ValueError, match="E4M3"):
        P.LinearWeights.from_row_major(u8(64, 96).view(dtype), u8(64, 3))


@pytest.mark.parametrize("dtype", OTHER_BYTES + [torch.float8_e4m3fn])
def test_scales_of_another_format_are_refused(dtype):
    u8 = lambda *s: torch.zeros(s, dtype=U8)  # noqa: E731
    refused(P.mxfp8_linear, (u8(4, 96), u8(4, 3).view(dtype)), weights())
    refused(P.mxfp8_linear, (u8(4, 96), u8(4, 3)), weights(), out=(u8(4, 64), u8(4, 2).view(dtype)))
    refused(P.mxfp8_quant, torch.zeros((4, 96), dtype=BF16), out=(u8(4, 96), u8(4, 3).view(dtype)))
    x, r, nw = norm_inputs()
    refused(P.add_rmsnorm_mxfp8, x, r, nw, out=P.TailOutput(None, u8(4, 64), u8(4, 2).view(dtype), None))
    with pytest.raises(ValueError, match="E8M0"):
        P.LinearWeights.from_row_major(u8(64, 96), u8(64, 3).view(dtype))


def test_bytes_and_their_own_formats_are_taken():
    u8 = lambda *s: torch.zeros(s, dtype=U8)  # noqa: E731
    own = lambda c, s: (c.view(torch.float8_e4m3fn), s.view(torch.float8_e8m0fnu))  # noqa: E731
    x = u8(4, 96), u8(4, 3)
    refused(P.mxfp8_linear, own(*x), weights(), out=own(u8(4, 64), u8(4, 2)), why="nothing is launched")
    refused(P.mxfp8_linear, x, weights(), out=(u8(4, 64), u8(4, 2)), why="nothing is launched")
    refused(P.mxfp8_quant, torch.zeros((4, 96), dtype=BF16), out=own(*x), why="nothing is launched")
    n, r, nw = norm_inputs()
    refused(P.add_rmsnorm_mxfp8, n, r, nw, out=P.TailOutput(None, *own(u8(4, 64), u8(4, 2)), None), why="nothing is launched")
