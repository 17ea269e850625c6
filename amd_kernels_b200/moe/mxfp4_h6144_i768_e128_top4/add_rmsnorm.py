"""Residual addition -> RMS norm -> MXFP8 and / or bf16 rows on B200, any row width, in one pass: what stands in front of the MoE layer
(behind the attention's output projection, at a model's first layer), where there are no slots for ``slots4_add_rmsnorm_mxfp8`` to
sum. Its MXFP8 rows are what ``mxfp8_linear`` and the shared expert read, its bf16 rows what ``mxfp4_moe`` reads."""
from __future__ import annotations

import torch

from ... import _lib
from .tail import TailOutput

MAX_H = 32768
_BF16, _U8 = torch.bfloat16, torch.uint8
CODE_DTYPES, SCALE_DTYPES = (torch.uint8, torch.float8_e4m3fn), (torch.uint8, torch.float8_e8m0fnu)


def row_stride(name, t, m, h, one_row=False):
    """The distance in elements of the rows of a [m, h] tensor that is not contiguous: unit stride along the row, a multiple of 8."""
    stride, unit = t.stride()
    if unit != 1:
        raise ValueError(f"{name}: expected unit stride along the row")
    if m > 1 and (stride & 7 or (stride < h and not (one_row and stride == 0))):
        raise ValueError(f"{name}: rows {stride} elements apart (needs a multiple of 8, at least {h})")
    return stride


def check_rows(name, t, shape, device):
    """bf16 [m, h] on CUDA device number ``device``; the distance of its rows in elements."""
    if t.dtype is not _BF16 or t.shape != shape or t.get_device() != device:
        raise ValueError(f"{name}: expected BF16 {list(shape)} on device {device}")
    return shape[1] if t.is_contiguous() else row_stride(name, t, *shape)


def check_mxfp8(name, codes, scales, m, width, device):
    """Contiguous [m, width] and [m, width / 32], uint8 or float8 of the two formats (E4M3FN, E8M0: a byte of another means another value)."""
    if codes is None or scales is None:
        raise ValueError(f"{name}: codes and scales come together")
    if (codes.dtype not in CODE_DTYPES or codes.shape != (m, width) or not codes.is_contiguous()
            or scales.dtype not in SCALE_DTYPES or scales.shape != (m, width // 32)
            or not scales.is_contiguous() or codes.get_device() != device or scales.get_device() != device):
        raise ValueError(f"{name}: expected contiguous codes [{m}, {width}] (uint8 or float8_e4m3fn) and scales [{m}, {width // 32}] "
                         f"(uint8 or float8_e8m0fnu) on device {device}")


def new_rows(m, width, dtype, like):
    """Contiguous [m, width] on the device of ``like`` (the strided form costs the interpreter half of what ``torch.empty`` costs)."""
    return torch.empty_strided((m, width), (width, 1), dtype=dtype, device=like.device)


def launch_on(device, call, *args):
    """``call(*args, stream)`` on the current stream of CUDA device number ``device``, which is made the current one where it is not."""
    if device < 0:
        raise ValueError("nothing is launched on tensors that are not on a CUDA device")
    if device == torch._C._cuda_getDevice():
        code = call(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            code = call(*args, torch._C._cuda_getCurrentRawStream(device))
    if code:
        _lib.check(code, call.__name__)


def add_rmsnorm_mxfp8(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-6, *,
                      weight_offset: float = 1.0, mxfp8: bool = True, bf16_out: bool = False,
                      out: TailOutput | None = None) -> TailOutput:
    """``s = x + residual`` in fp32 (residual out ``bf16(s)``), ``y = s * rstd * (weight + weight_offset)``, MXFP8 of the fp32 ``y``
    and / or ``bf16(y)``: steps 2-4 of ``amd_kernels/norm/gemma_add_rmsnorm_h6144/reference.py`` (whose weight offset is 1; 0 is
    the plain RMS norm) at any width H that is a multiple of 32, up to 32768.

    ``x`` and ``residual`` bf16 [M, H], rows any multiple of 8 elements apart; M may be 0. ``residual`` None: ``s = x``, and no residual
    comes back. A residual expanded from one row (stride 0) is added to every row. ``out``: where the results go; its tensors
    that are not None say what is computed (``mxfp8`` and ``bf16_out`` are not read). Its ``residual`` and ``normed`` may be ``x`` or
    ``residual`` itself; codes and scales are contiguous. A row's bits depend on nothing but the row."""
    shape, device = x.shape, x.get_device()
    if x.dtype is not _BF16 or len(shape) != 2:
        raise ValueError("expected BF16 [M, H] rows")
    m, h = shape
    if h < 32 or h % 32 or h > MAX_H:
        raise ValueError(f"rows of {h} columns (needs a multiple of 32, up to {MAX_H})")
    xs = h if x.is_contiguous() else row_stride("x", x, m, h)
    r_at = rs = ro_at = n_at = c_at = s_at = 0
    ros = ns = h
    if residual is not None:
        if residual.dtype is not _BF16 or residual.shape != shape or residual.get_device() != device:
            raise ValueError(f"residual: expected BF16 [{m}, {h}] on device {device}")
        rs = h if residual.is_contiguous() else row_stride("residual", residual, m, h, True)
        r_at = residual.data_ptr()
    if weight.dtype is not _BF16 or weight.shape != (h,) or not weight.is_contiguous() or weight.get_device() != device:
        raise ValueError(f"weight: expected contiguous BF16 [{h}] on device {device}")
    if out is None:
        ro = codes = scales = normed = None
        if residual is not None:
            ro = new_rows(m, h, _BF16, x)
            ro_at = ro.data_ptr()
        if mxfp8:
            codes, scales = new_rows(m, h, _U8, x), new_rows(m, h // 32, _U8, x)
            c_at, s_at = codes.data_ptr(), scales.data_ptr()
        elif not bf16_out and ro is None:
            raise ValueError("no output asked for")
        if bf16_out:
            normed = new_rows(m, h, _BF16, x)
            n_at = normed.data_ptr()
        out = TailOutput(ro, codes, scales, normed)
    else:
        ro, codes, scales, normed = out.residual, out.codes, out.scales, out.normed
        if ro is not None:
            if residual is None:
                raise ValueError("out.residual without a residual")
            ros = check_rows("out.residual", ro, shape, device)
            ro_at = ro.data_ptr()
        if normed is not None:
            ns = check_rows("out.normed", normed, shape, device)
            n_at = normed.data_ptr()
        if codes is not None or scales is not None:
            check_mxfp8("out", codes, scales, m, h, device)
            c_at, s_at = codes.data_ptr(), scales.data_ptr()
        elif ro is None and normed is None:
            raise ValueError("no output asked for")
    launch_on(device, _lib.load().b200moe_add_rmsnorm_quant, _lib.NORM_CALL.pack(
        x.data_ptr(), xs, r_at, rs, weight.data_ptr(), ro_at, ros, n_at, ns, c_at, s_at, m, h, weight_offset, eps))
    return out
