"""The MXFP8 matrix product with bias, activation and residual in its epilogue on B200: the projections around the MoE layer. It reads
the MXFP8 rows that ``slots4_add_rmsnorm_mxfp8`` and ``add_rmsnorm_mxfp8`` hand out (or quantises bf16 rows itself) and writes bf16
rows, added to the residual stream if asked, or MXFP8 rows for the next product. E4M3 codes with one E8M0 scale per 32 elements
on both sides, fp32 accumulation; the shared expert (``SharedWeights``) is two such products of fixed shape."""
from __future__ import annotations

from dataclasses import dataclass

import torch

from ... import _lib
from .add_rmsnorm import CODE_DTYPES, SCALE_DTYPES, check_mxfp8, check_rows, launch_on, new_rows, row_stride
from .chain import status_word

MAX_DIM, MAX_ROWS = 1 << 20, 1 << 24
ROWS_INSIDE = 64  # up to so many bf16 rows are quantised inside the product's launch


@dataclass
class LinearWeights:
    """A weight [rows, k] in the kernels' layout, built once by ``from_row_major`` before graph capture. ``tiles`` u8: [row tile][K-tile]
    images of 128 rows x 128 K-elements of E4M3 codes as the 128-byte swizzle lays them in shared memory, then the tiles' scale
    atoms. ``bias`` fp32 [rows] or None."""
    tiles: torch.Tensor
    bias: torch.Tensor | None
    rows: int
    k: int
    gated: bool

    @property
    def n(self) -> int:
        """Output columns."""
        return self.rows // 2 if self.gated else self.rows

    @classmethod
    def from_row_major(cls, w, scale, bias=None, *, gated: bool = False):
        """From row-major E4M3 codes [rows, K] (uint8 or float8_e4m3fn), E8M0 scales [rows, K / 32] (uint8 or float8_e8m0fnu) and a bias
        [rows] of any floating type. K a multiple of 32, rows a multiple of 8. ``gated``: the first half of the rows are the gate,
        the second half the up projection (each a multiple of 32); the activation of the call is then a gated one."""
        if w.ndim != 2 or w.dtype not in CODE_DTYPES or scale.dtype not in SCALE_DTYPES:
            raise ValueError("expected E4M3 codes [rows, K] (uint8 or float8_e4m3fn) and E8M0 scales [rows, K / 32] (uint8 or float8_e8m0fnu)")
        rows, k = w.shape
        if not w.is_cuda or scale.device != w.device or (bias is not None and bias.device != w.device):
            raise ValueError("weights must be CUDA tensors of one device")
        nbytes = int(_lib.load().b200moe_linear_weight_bytes(rows, k, int(gated)))
        if nbytes == 0:
            raise ValueError(f"unsupported weight [{rows}, {k}]: K a multiple of 32, rows a multiple of {64 if gated else 8}, both up to {MAX_DIM}")
        if scale.shape != (rows, k // 32):
            raise ValueError(f"scales: needs [{rows}, {k // 32}]")
        if bias is not None:
            if bias.shape != (rows,) or not bias.is_floating_point():
                raise ValueError(f"bias: needs [{rows}] of a floating type")
            bias = bias.detach().float().contiguous()
            if bias.data_ptr() & 15:
                bias = bias.clone()
        codes, scales = w.contiguous().view(torch.uint8), scale.contiguous().view(torch.uint8)
        if codes.data_ptr() & 15:
            codes = codes.clone()
        tiles = torch.empty(nbytes, dtype=torch.uint8, device=w.device)
        launch_on(w.get_device(), _lib.load().b200moe_preshuffle_linear, codes.data_ptr(), scales.data_ptr(), rows, k, int(gated),
                  tiles.data_ptr())
        return cls(tiles, bias, rows, k, bool(gated))


def mxfp8_quant(x: torch.Tensor, *, out=None):
    """bf16 [M, K] -> (E4M3 codes u8 [M, K], E8M0 scales u8 [M, K / 32]): ``shared_quant_rows`` at any width that is a multiple of 32
    (the same bits at 6144; an infinite value saturates and keeps its block's scale finite). Rows any multiple of 8 elements apart."""
    if x.ndim != 2 or x.dtype is not torch.bfloat16:
        raise ValueError("expected BF16 [M, K]")
    m, k = x.shape
    device = x.get_device()
    if k < 32 or k % 32 or k > MAX_DIM or m > MAX_ROWS:
        raise ValueError(f"rows of {k} columns (needs a multiple of 32, up to {MAX_DIM}; up to {MAX_ROWS} rows)")
    stride = k if x.is_contiguous() else row_stride("x", x, m, k, True)
    if out is None:
        out = new_rows(m, k, torch.uint8, x), new_rows(m, k // 32, torch.uint8, x)
    else:
        check_mxfp8("out", *out, m, k, device)
    launch_on(device, _lib.load().b200moe_quant_mxfp8, x.data_ptr(), stride, m, k, out[0].data_ptr(), out[1].data_ptr())
    return out


def mxfp8_linear(x, w: LinearWeights, *, activation: str | None = None, residual: torch.Tensor | None = None,
                 mxfp8_out: bool = False, out=None):
    """``y = activation(x @ w.T + bias) + residual``, fp32 until one rounding at the end.

    ``x``: MXFP8 rows as a pair (codes [M, K], scales [M, K / 32]), or bf16 [M, K], quantised as by
    ``mxfp8_quant`` (up to 64 rows inside the product's launch, more in one in front of it; the same bits). M may be 0. Rows
    for weights wider than some 6144 x 6144, rows that several products read, and most captured calls are faster quantised once
    with ``mxfp8_quant``.
    ``activation``: None, "relu", "silu", "gelu" (exact), "gelu_tanh"; for gated weights "swiglu" (silu(gate) * up) or "swiglu_oai"
    (the MoE layer's: clamped, alpha 1.702, up + 1). ``residual`` bf16 [M, N], rows any multiple of 8 elements apart.
    Returns bf16 [M, N], or with ``mxfp8_out`` the pair (codes [M, N], scales [M, N / 32]) that the next product reads.
    ``out``: where the result goes, a bf16 tensor or a pair (``mxfp8_out`` is then not read); a bf16 ``out`` may be the residual
    itself, and nothing else that the call reads. The sums of one call repeat bit for bit; between calls of different M they may be
    split along K in another way."""
    act = _lib.ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r}")
    if (act >= 5) != w.gated:
        raise ValueError(f"activation {activation!r} on {'gated' if w.gated else 'plain'} weights")
    tiles, bias, rows, k, gated = w.tiles, w.bias, w.rows, w.k, w.gated
    n, device = rows // 2 if gated else rows, tiles.get_device()
    x_at = xs = r_at = rs = y_at = oc_at = os_at = 0
    ys = n
    if isinstance(x, torch.Tensor):
        if x.dtype is not torch.bfloat16 or x.ndim != 2 or x.shape[1] != k or x.get_device() != device:
            raise ValueError(f"x: expected BF16 [M, {k}] (or a pair of codes and scales) on device {device}")
        m = x.shape[0]
        xs, x_at = k if x.is_contiguous() else row_stride("x", x, m, k, True), x.data_ptr()
        c_at = s_at = 0
        if m > ROWS_INSIDE:
            quantised = tiles.new_empty(m * (k + k // 32))
            c_at = quantised.data_ptr()
            s_at = c_at + m * k
    elif isinstance(x, (tuple, list)) and len(x) == 2 and x[0] is not None:
        codes, scales = x
        m = codes.shape[0] if codes.ndim else 0
        check_mxfp8("x", codes, scales, m, k, device)
        c_at, s_at = codes.data_ptr(), scales.data_ptr()
    else:
        raise ValueError("expected BF16 [M, K] rows or a pair of codes and scales")
    if residual is not None:
        rs, r_at = check_rows("residual", residual, (m, n), device), residual.data_ptr()
    if out is None:
        if mxfp8_out:
            if n % 32:
                raise ValueError(f"MXFP8 output of {n} columns (needs a multiple of 32)")
            out = new_rows(m, n, torch.uint8, tiles), new_rows(m, n // 32, torch.uint8, tiles)
            oc_at, os_at = out[0].data_ptr(), out[1].data_ptr()
        else:
            out = new_rows(m, n, torch.bfloat16, tiles)
            y_at = out.data_ptr()
    elif isinstance(out, torch.Tensor):
        ys, y_at = check_rows("out", out, (m, n), device), out.data_ptr()
    else:
        if n % 32:
            raise ValueError(f"MXFP8 output of {n} columns (needs a multiple of 32)")
        check_mxfp8("out", *out, m, n, device)
        oc_at, os_at = out[0].data_ptr(), out[1].data_ptr()
    status = status_word(tiles.device).data_ptr() if device >= 0 else 0
    launch_on(device, _lib.load().b200moe_linear, _lib.LINEAR_CALL.pack(
        tiles.data_ptr(), 0 if bias is None else bias.data_ptr(), rows, k, gated, x_at, xs, c_at, s_at, m, r_at, rs, y_at, ys, oc_at,
        os_at, act), status)
    return out
