"""Residual addition -> RMS norm -> MXFP8 and / or bf16 rows on B200, any row width, in one pass: what stands in front of the MoE layer
(behind the attention's output projection, at a model's first layer), where there are no slots for ``slots4_add_rmsnorm_mxfp8`` to
sum. Its MXFP8 rows are what ``mxfp8_linear`` and the shared expert read, its bf16 rows what ``mxfp4_moe`` reads."""
from __future__ import annotations

import torch

from ... import _lib
from .tail import TailOutput

MAX_H = 65536
_BF16 = torch.bfloat16


def rows_of(name, t, m, h, dev, shared_row=False):
    """Checks bf16 rows [m, h] with unit column stride, a multiple of 8 elements apart; that distance."""
    if t.dtype is not _BF16 or t.shape != (m, h) or t.device != dev:
        raise ValueError(f"{name}: expected BF16 [{m}, {h}] on {dev}")
    stride, unit = t.stride()
    if unit != 1:
        raise ValueError(f"{name}: expected unit stride along the row")
    if m > 1 and (stride & 7 or (stride < h and not (shared_row and stride == 0))):
        raise ValueError(f"{name}: rows {stride} elements apart (needs a multiple of 8, at least {h})")
    return stride


def check_mxfp8(name, codes, scales, m, width, dev):
    """Contiguous [m, width] and [m, width / 32] of one byte each (uint8, or float8 of the two formats)."""
    if codes is None or scales is None:
        raise ValueError(f"{name}: codes and scales come together")
    if (codes.element_size() != 1 or codes.shape != (m, width) or not codes.is_contiguous() or codes.device != dev
            or scales.element_size() != 1 or scales.shape != (m, width // 32) or not scales.is_contiguous() or scales.device != dev):
        raise ValueError(f"{name}: expected contiguous codes [{m}, {width}] and scales [{m}, {width // 32}] of one byte each on {dev}")


def launch_on(dev, call, *args):
    """``call(*args, stream)`` on the current stream of ``dev``, which is made the current device where it is not. A device that is no
    CUDA device is a ValueError."""
    if dev.type != "cuda":
        raise ValueError(f"expected tensors on a CUDA device, got {dev}")
    if dev.index == torch._C._cuda_getDevice():
        code = call(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            code = call(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if code:
        _lib.check(code, call.__name__)


def add_rmsnorm_mxfp8(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-6, *,
                      weight_offset: float = 1.0, mxfp8: bool = True, bf16_out: bool = False,
                      out: TailOutput | None = None) -> TailOutput:
    """``s = x + residual`` in fp32 (residual out ``bf16(s)``), ``y = s * rstd * (weight + weight_offset)``, MXFP8 of the fp32 ``y``
    and / or ``bf16(y)``: steps 2-4 of ``amd_kernels/norm/gemma_add_rmsnorm_h6144/reference.py`` (whose weight offset is 1; 0 is
    the plain RMS norm) at any width H that is a multiple of 32, up to 65536.

    ``x`` and ``residual`` bf16 [M, H], rows any multiple of 8 elements apart; M may be 0. ``residual`` None: ``s = x``, and no residual
    comes back. A residual expanded from one row (stride 0) is added to every row. ``out``: where the results go; its tensors
    that are not None say what is computed (``mxfp8`` and ``bf16_out`` are not read). Its ``residual`` and ``normed`` may be ``x`` or
    ``residual`` itself; codes and scales are contiguous. A row's bits depend on nothing but the row."""
    if x.ndim != 2 or weight.ndim != 1:
        raise ValueError("expected BF16 [M, H] rows and a [H] weight")
    m, h = x.shape
    dev = x.device
    if h < 32 or h % 32 or h > MAX_H:
        raise ValueError(f"rows of {h} columns (needs a multiple of 32, up to {MAX_H})")
    xs = rows_of("x", x, m, h, dev)
    rs = 0 if residual is None else rows_of("residual", residual, m, h, dev, True)
    if weight.dtype is not _BF16 or weight.shape != (h,) or not weight.is_contiguous() or weight.device != dev:
        raise ValueError(f"weight: expected contiguous BF16 [{h}] on {dev}")
    ros = ns = h
    if out is None:
        empty = torch.empty
        out = TailOutput(None if residual is None else empty((m, h), dtype=_BF16, device=dev),
                         empty((m, h), dtype=torch.uint8, device=dev) if mxfp8 else None,
                         empty((m, h // 32), dtype=torch.uint8, device=dev) if mxfp8 else None,
                         empty((m, h), dtype=_BF16, device=dev) if bf16_out else None)
        ro, codes, scales, normed = out.residual, out.codes, out.scales, out.normed
    else:
        ro, codes, scales, normed = out.residual, out.codes, out.scales, out.normed
        if ro is not None:
            if residual is None:
                raise ValueError("out.residual without a residual")
            ros = rows_of("out.residual", ro, m, h, dev)
        if normed is not None:
            ns = rows_of("out.normed", normed, m, h, dev)
        if codes is not None or scales is not None:
            check_mxfp8("out", codes, scales, m, h, dev)
    if ro is None and normed is None and codes is None:
        raise ValueError("no output asked for")
    call = _lib.NORM_CALL.pack(x.data_ptr(), xs, 0 if residual is None else residual.data_ptr(), rs, weight.data_ptr(),
                               0 if ro is None else ro.data_ptr(), ros, 0 if normed is None else normed.data_ptr(), ns,
                               0 if codes is None else codes.data_ptr(), 0 if scales is None else scales.data_ptr(), m, h,
                               weight_offset, eps)
    launch_on(dev, _lib.load().b200moe_add_rmsnorm_quant, call)
    return out
