"""Residual RMS norm over partial sums, its 8-bit output and its gradient (``native/hip/norm.hip``).

A tensor-parallel layer ends with a sum over ranks, the residual stream's addition and a norm in
front of the next product.  :func:`add_rms_norm` does all three in one pass over 1..8 partial sums
(``XgmiAllReduce.all_reduce_norm`` calls it on the peers' buffers)::

    h            = sum(srcs) + residual               # fp32, in list order, the residual last
    residual_out = round(h)
    rstd         = 1 / sqrt(mean(h**2) + eps)         # over the last dimension
    out          = round(h * rstd * weight)           # or e4m3 codes and scales

Every entry point runs on the tensors' device and that device's current stream, writes into tensors
that the caller allocated, and raises if the library is missing.  Nothing is synchronised, allocated
on the host or kept between calls, so the calls can be captured into a graph.

None is part of an autograd graph: with grad mode on, tensors that require grad are refused.  In an
``autograd.Function`` the first is the forward pass and the second the backward one.
"""

from __future__ import annotations

import struct
from operator import methodcaller

from . import hip

MAX_SRCS = 8
MAX_COLS = 32768  # a row stays in the registers of one workgroup
GROUP = 128  # columns that share a scale

# native/hip/norm.hip:NormParams and NormBackwardParams
_FORWARD = struct.Struct("=9Q9q" + "QQqQqQQQ" + "6ifi")
_BACKWARD = struct.Struct("=QqQqQqQQQqQQQ" + "6i")
_OVERLAP = -1
_NO_INPUTS = [0] * (MAX_SRCS + 1)


def _kinds():
    """Type codes and e4m3, once torch is there (the package is imported without it too)."""
    global _KINDS
    import torch

    _KINDS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}, torch.float32, torch.float8_e4m3fn
    return _KINDS


_KINDS = None


def _pitch(t, shape, dtype, what, written=False):
    """The row stride of ``t`` in elements, after its checks."""
    if t.dtype is not dtype:
        raise ValueError(f"{what}: expected {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    cols = shape[-1]
    if len(shape) != 2:
        if not t.is_contiguous():
            raise ValueError(f"{what}: only 2-D tensors may have strides")
        return cols
    pitch, inner = t.stride()
    if inner != 1 and cols > 1:
        raise ValueError(f"{what}: the last dimension must be contiguous")
    if written and pitch < cols and shape[0] > 1:
        raise ValueError(f"{what}: its rows overlap")
    return pitch


def _flat(t, shape, dtype, other, what):
    if t.dtype is not dtype and t.dtype is not other:
        raise ValueError(f"{what}: expected {dtype}{'' if other is dtype else f' or {other}'}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: must be contiguous")


_device = methodcaller("get_device")


def _on_one_device(device, tensors):
    if device < 0 or set(map(_device, tensors)) != {device}:
        raise ValueError("every tensor must be on one CUDA device")


def _failed(rc, what):
    if rc == _OVERLAP:
        raise ValueError("an output overlaps another tensor of the call (an output may replace an input of its type "
                         "element on element, and nothing else)")
    hip._check(rc, what)


def add_rms_norm(srcs, weight, out, *, residual=None, residual_out=None, rstd=None, scales=None, eps=1e-6) -> None:
    """The sum of 1..8 partial sums and the residual, normalised over the last dimension.

    ``srcs`` (a list), ``residual`` and ``residual_out`` have ``out``'s shape ``(..., cols)`` with
    ``cols`` up to 32768, and one type: fp32, bf16 or fp16.  2-D tensors may have any row stride (a
    residual or partial sum with stride 0 is one row for all), others are contiguous.  ``weight``:
    ``(cols,)`` of that type or fp32.

    ``residual_out``, where given, takes the rounded sum, the next layer's residual and what the
    backward pass needs; ``rstd`` (fp32, shape ``(...)``) the reciprocal root mean square.  Either
    and ``out`` may be one of the inputs itself (same memory, same strides), no other overlap.

    ``out`` has the inputs' type, or is ``float8_e4m3fn`` with ``scales`` (fp32): of shape ``(...)``
    for one scale a row, or ``(..., ceil(cols / 128))`` for one a group of 128 columns.  A scale is
    the largest magnitude / 448 (zero, with all codes zero, where the magnitude is below 2**-100); a code
    is the value times the scale's reciprocal, both in fp32, rounded to nearest even; ``code * scale`` is
    the value.

    Sums and statistics are fp32; ``out`` comes from the unrounded sum and is rounded once.  An
    infinity or NaN in a row makes that row (in 8 bits: its scale) NaN or infinite and no other.  A row
    whose squares add up to more than fp32 holds (a root mean square of 1.8e19 / sqrt(cols)) has ``rstd``
    and ``out`` zero.  With ``eps`` zero, squares below 1e-38 lose their precision (a root mean square of
    1e-19), and a row of zeros is NaN.
    """
    args = _arguments(srcs, weight, out, residual, residual_out, rstd, scales, eps)
    if args:
        _launch(*args)
        hip._written([t for t in (out, residual_out, rstd, scales) if t is not None])


def _arguments(srcs, weight, out, residual, residual_out, rstd, scales, eps):
    """:func:`_launch`'s arguments, after every check; ``None`` without rows."""
    kinds, f32, e4m3 = _KINDS or _kinds()
    if not 1 <= len(srcs) <= MAX_SRCS:
        raise ValueError(f"1..{MAX_SRCS} partial sums")
    dtype, shape, device = srcs[0].dtype, out.shape, out.get_device()
    if dtype not in kinds:
        raise ValueError(f"partial sums: expected fp32, bf16 or fp16, got {dtype}")
    if not shape or not 1 <= shape[-1] <= MAX_COLS:
        raise ValueError(f"out: expected (..., cols) with 1..{MAX_COLS} columns, got shape {tuple(shape)}")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    cols, leading = shape[-1], shape[:-1]
    kind = scales_ptr = h_ptr = h_pitch = rstd_ptr = 0
    if out.dtype is e4m3:
        if scales is None:
            raise ValueError("an e4m3 output needs scales")
        kind = 1 if scales.dim() == len(leading) else 2
        _flat(scales, leading if kind == 1 else leading + (-(-cols // GROUP),), f32, f32, "scales")
        scales_ptr = scales.data_ptr()
    elif scales is not None:
        raise ValueError("scales belong to an e4m3 output")
    out_pitch = _pitch(out, shape, e4m3 if kind else dtype, "out", True)
    tensors = [*srcs, weight, out]
    first, strides = _pitch(srcs[0], shape, dtype, "partial sum"), srcs[0].stride()
    pitches = [first, *[first if t.dtype is dtype and t.shape == shape and t.stride() == strides else
                        _pitch(t, shape, dtype, "partial sum") for t in srcs[1:]]]  # most are alike
    ptrs = [t.data_ptr() for t in srcs]
    if residual is not None:
        pitches.append(first if residual.dtype is dtype and residual.shape == shape and residual.stride() == strides else
                       _pitch(residual, shape, dtype, "residual"))
        ptrs.append(residual.data_ptr())
        tensors.append(residual)
    if residual_out is not None:
        h_pitch, h_ptr = _pitch(residual_out, shape, dtype, "residual_out", True), residual_out.data_ptr()
        tensors.append(residual_out)
    _flat(weight, (cols,), dtype, f32, "weight")
    if rstd is not None:
        _flat(rstd, leading, f32, f32, "rstd")
        rstd_ptr = rstd.data_ptr()
        tensors.append(rstd)
    if scales_ptr:
        tensors.append(scales)
    hip._refuse_grad(tensors)
    _on_one_device(device, tensors)
    rows = out.numel() // cols
    if not rows:
        return None
    return (ptrs, pitches, weight.data_ptr(), out.data_ptr(), out_pitch, h_ptr, h_pitch, rstd_ptr, scales_ptr, rows, cols,
            kinds[dtype], weight.dtype is f32, kind, device, eps)


def _launch(ptrs, pitches, weight, out, out_pitch, h, h_pitch, rstd, scales, rows, cols, dtype, weight_f32, kind, device,
            eps):
    """The call into the library, on addresses (inputs may be a peer's memory)."""
    n = len(ptrs)
    pad = _NO_INPUTS[n:]
    block = _FORWARD.pack(*ptrs, *pad, *pitches, *pad, weight, out, out_pitch, h, h_pitch, rstd, scales, rows, cols, n,
                          dtype, weight_f32, kind, device, eps, 0)
    rc = (hip._lib or hip.lib()).netop_add_rms_norm(block, hip._raw_stream(device))
    if rc:
        _failed(rc, "netop_add_rms_norm")


def add_rms_norm_backward(dy, h, weight, rstd, dh, dweight, *, dresidual=None) -> None:
    """The gradient of :func:`add_rms_norm` (with an output of the inputs' type).

    ``h`` is its ``residual_out`` and ``rstd`` its ``rstd``; ``dy`` the gradient of ``out``,
    ``dresidual``, where given, that of ``residual_out``.  ``dh`` takes the gradient of the sum, which
    is that of each partial sum and of the residual (for one that was a row for all: its rows' sum),
    and may be ``dy``, ``h`` or ``dresidual`` itself.  It is right for rows of any magnitude that the forward
    pass takes; where ``rstd`` is zero it is ``dresidual``.  ``dweight`` (``(cols,)``, the weight's type or
    fp32) takes the weight's gradient, summed over the rows in fp32 in an order that depends on the
    shape alone: the same inputs give the same bits.
    """
    import torch

    kinds, f32, _ = _KINDS or _kinds()
    dtype, shape, device = dy.dtype, dy.shape, dy.get_device()
    if dtype not in kinds:
        raise ValueError(f"dy: expected fp32, bf16 or fp16, got {dtype}")
    if not shape or not 1 <= shape[-1] <= MAX_COLS:
        raise ValueError(f"dy: expected (..., cols) with 1..{MAX_COLS} columns, got shape {tuple(shape)}")
    cols = shape[-1]
    rows = dy.numel() // cols
    dy_pitch = _pitch(dy, shape, dtype, "dy")
    h_pitch = _pitch(h, shape, dtype, "h")
    dh_pitch = _pitch(dh, shape, dtype, "dh", True)
    dres_pitch = 0 if dresidual is None else _pitch(dresidual, shape, dtype, "dresidual")
    _flat(weight, (cols,), dtype, f32, "weight")
    _flat(rstd, shape[:-1], f32, f32, "rstd")
    _flat(dweight, (cols,), weight.dtype, f32, "dweight")
    tensors = [dy, h, weight, rstd, dh, dweight]
    if dresidual is not None:
        tensors.append(dresidual)
    hip._refuse_grad(tensors)
    _on_one_device(device, tensors)
    L = hip._lib or hip.lib()
    parts = L.netop_norm_backward_parts(rows, cols)
    partial = torch.empty(parts * cols, dtype=f32, device=dy.device)
    block = _BACKWARD.pack(dy.data_ptr(), dy_pitch, h.data_ptr(), h_pitch,
                           0 if dresidual is None else dresidual.data_ptr(), dres_pitch, weight.data_ptr(),
                           rstd.data_ptr(), dh.data_ptr(), dh_pitch, dweight.data_ptr(), partial.data_ptr(), rows,
                           cols, parts, kinds[dtype], weight.dtype is f32, dweight.dtype is f32, device)
    rc = L.netop_add_rms_norm_backward(block, hip._raw_stream(device))
    if rc:
        _failed(rc, "netop_add_rms_norm_backward")
    hip._written((dh, dweight))
