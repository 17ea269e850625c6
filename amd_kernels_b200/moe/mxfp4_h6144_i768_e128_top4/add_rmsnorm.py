"""Residual addition -> RMS norm -> MXFP8 and / or bf16 rows on B200, any row width, in one pass: what stands in front of the MoE layer
(behind the attention's output projection, at a model's first layer), where there are no slots for ``slots4_add_rmsnorm_mxfp8`` to
sum. Its MXFP8 rows are what ``mxfp8_linear`` and the shared expert read, its bf16 rows what ``mxfp4_moe`` reads."""
from __future__ import annotations

import torch

from ... import _lib
from .chain import _raw_stream
from .tail import TailOutput

MAX_H = 65536


def _rows(name, t, m, h, dev, shared_row=False):
    """Checks bf16 rows [m, h] with unit column stride and 16-byte aligned rows; their stride in elements."""
    if t.dtype != torch.bfloat16 or t.shape != (m, h) or t.stride(1) != 1 or t.device != dev:
        raise ValueError(f"{name}: expected BF16 [{m}, {h}] with unit stride along the row, on {dev}")
    stride = t.stride(0)
    if m > 1 and (stride & 7 or (stride < h and not (shared_row and stride == 0))):
        raise ValueError(f"{name}: rows {stride} elements apart (needs a multiple of 8, at least {h})")
    return stride


def add_rmsnorm_mxfp8(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-6, *,
                      weight_offset: float = 1.0, mxfp8: bool = True, bf16_out: bool = False,
                      out: TailOutput | None = None) -> TailOutput:
    """``s = x + residual`` in fp32 (residual out ``bf16(s)``), ``y = s * rstd * (weight + weight_offset)``, MXFP8 of the fp32 ``y``
    and / or ``bf16(y)``: steps 2-4 of ``amd_kernels/norm/gemma_add_rmsnorm_h6144/reference.py`` (whose weight offset is 1; 0 is
    the plain RMS norm) at any width H that is a multiple of 32, up to 65536.

    ``x`` and ``residual`` bf16 [M, H], rows any multiple of 8 elements apart; M may be 0. ``residual`` None: ``s = x``, and no residual
    comes back. A residual expanded from one row (stride 0) is added to every row. ``out``: where the results go; its tensors
    that are not None say what is computed (``mxfp8`` and ``bf16_out`` are not read). Its ``residual`` may be ``residual`` or ``x``
    itself, its ``normed`` ``x``; codes and scales are contiguous. A row's bits depend on nothing but the row."""
    if x.ndim != 2 or weight.ndim != 1:
        raise ValueError("expected BF16 [M, H] rows and a [H] weight")
    (m, h), dev = x.shape, x.device
    if h < 32 or h % 32 or h > MAX_H:
        raise ValueError(f"rows of {h} columns (needs a multiple of 32, up to {MAX_H})")
    xs = _rows("x", x, m, h, dev)
    rs = 0 if residual is None else _rows("residual", residual, m, h, dev, shared_row=True)
    if weight.dtype != torch.bfloat16 or weight.shape[0] != h or not weight.is_contiguous() or weight.device != dev:
        raise ValueError(f"weight: expected contiguous BF16 [{h}] on {dev}")
    ros = ns = h
    if out is None:
        empty = torch.empty
        out = TailOutput(None if residual is None else empty((m, h), dtype=torch.bfloat16, device=dev),
                         empty((m, h), dtype=torch.uint8, device=dev) if mxfp8 else None,
                         empty((m, h // 32), dtype=torch.uint8, device=dev) if mxfp8 else None,
                         empty((m, h), dtype=torch.bfloat16, device=dev) if bf16_out else None)
        if residual is None and not mxfp8 and not bf16_out:
            raise ValueError("no output asked for")
    else:
        if out.residual is not None:
            if residual is None:
                raise ValueError("out.residual without a residual")
            ros = _rows("out.residual", out.residual, m, h, dev)
        if out.normed is not None:
            ns = _rows("out.normed", out.normed, m, h, dev)
        if out.codes is not None or out.scales is not None:
            check_mxfp8("out", out.codes, out.scales, m, h, dev)
        if out.residual is None and out.normed is None and out.codes is None:
            raise ValueError("no output asked for")
    call = _lib.load().b200moe_add_rmsnorm_quant
    args = (x.data_ptr(), xs, None if residual is None else residual.data_ptr(), rs, weight.data_ptr(), weight_offset, eps, m, h,
            None if out.residual is None else out.residual.data_ptr(), ros, None if out.normed is None else out.normed.data_ptr(), ns,
            None if out.codes is None else out.codes.data_ptr(), None if out.scales is None else out.scales.data_ptr())
    launch_on(dev, call, args, "add_rmsnorm_quant")
    return out


def check_mxfp8(name, codes, scales, m, width, dev):
    """Contiguous uint8 (or float8 of the two formats) [m, width], [m, width / 32]."""
    if codes is None or scales is None:
        raise ValueError(f"{name}: codes and scales come together")
    if (codes.element_size() != 1 or codes.shape != (m, width) or not codes.is_contiguous() or codes.device != dev
            or scales.element_size() != 1 or scales.shape != (m, width // 32) or not scales.is_contiguous() or scales.device != dev):
        raise ValueError(f"{name}: expected contiguous codes [{m}, {width}] and scales [{m}, {width // 32}] of one byte each on {dev}")


def launch_on(dev, call, args, what):
    """``call(*args, stream)`` on the current stream of ``dev``, which is made the current device where it is not."""
    stream = _raw_stream(dev)
    if dev.index == torch.cuda.current_device():
        code = call(*args, stream)
    else:
        with torch.cuda.device(dev):
            code = call(*args, stream)
    if code:
        _lib.check(code, what)
