"""The decoder layer's RMS norm on MI355X, with the residual's addition in front
of it and, for fp8_block projections behind it, its result in e4m3 codes.

The reference norms the stream in front of each layer and adds the layer's
result to it (``src/mlx_lean_moe/model/qwen3_5/transformer.py:110-112``):
``h = rows + attention(rms_norm(rows))``. :func:`rms_norm` is that norm over one
pass of memory, the addition of the layer before it included.
"""

from __future__ import annotations

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .gated_delta import _FLOATS, _require_device, _stream
from .quant import QuantizedRows, _followed, rows_overlap

_F32 = torch.float32


def _row_layout(t: torch.Tensor, K: int) -> int:
    """Elements between the rows of K that ``t`` consists of, 0 if they do not lie
    evenly apart."""

    if t.is_contiguous():
        return K
    if t.ndim == 2 and (t.stride(1) == 1 or K == 1) and t.stride(0) >= K:
        return t.stride(0)
    return 0


def _new_rows(x: torch.Tensor) -> torch.Tensor:
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None, eps: float, *, residual: torch.Tensor | None = None,
             quantize: bool = False, keep_rows: bool = False, sum_out: torch.Tensor | None = None):
    """``s * weight / sqrt(mean(s * s) + eps)`` over the last axis, ``s = x``, or
    ``x + residual`` rounded to their dtype.

    ``x`` and ``residual (..., K)`` of one float dtype (rows at any stride, e.g.
    column slices); ``weight (K,)`` or None (ones). The result is formed in 64 bits
    and rounded to float32 and then to x's dtype; it does not depend on the other rows.

    Without a residual the normed rows are returned, with one ``(normed, s)``:
    ``s`` is the stream that the next layer's result is added to, written to
    ``sum_out`` if given, which may be ``x`` or ``residual`` itself and must not
    overlap them otherwise.

    ``quantize=True`` gives the normed rows as :class:`QuantizedRows` (K a multiple
    of 16): the codes that an fp8_block product would make of them, and with
    ``keep_rows=True`` the rows as well. No gradient: a tensor that needs one, or
    that forward mode follows, raises ``RuntimeError``."""

    if x.ndim == 0 or x.shape[-1] == 0:
        raise ValueError("rms_norm takes rows of at least one value")
    K, dtype = x.shape[-1], x.dtype
    index = x.get_device()
    if index < 0 or dtype not in _FLOATS:
        _require_device(x)
    if weight is not None:
        if weight.shape != (K,):
            raise ValueError(f"weight must have shape ({K},), got {tuple(weight.shape)}")
        if weight.get_device() != index or weight.dtype not in _FLOATS:
            _require_device(x, weight)
        if weight.dtype is not _F32 or not weight.is_contiguous():
            weight = weight.float().contiguous()
    if residual is None:
        if sum_out is not None:
            raise ValueError("sum_out goes with a residual")
    elif residual.shape != x.shape or residual.dtype is not dtype:
        raise ValueError(f"residual must be {tuple(x.shape)} {dtype}, got {tuple(residual.shape)} {residual.dtype}")
    elif residual.get_device() != index:
        _require_device(x, residual)
    if keep_rows and not quantize:
        raise ValueError("keep_rows goes with quantize")
    if quantize and K % 16:
        raise ValueError(f"quantized rows have a multiple of 16 values, got {K}")
    if _followed(x, weight, residual, sum_out):
        raise RuntimeError("rms_norm has no gradient and no forward mode; call it under torch.no_grad()")
    device, given = x.device, sum_out is not None
    M = x.numel() // K
    x_stride = _row_layout(x, K)
    if not x_stride:
        x, x_stride = x.contiguous(), K
    # (a third of torch.empty's time, and a norm of few rows is host-bound)
    new = torch.empty_like if x.is_contiguous() else _new_rows
    r_stride = s_stride = K
    if residual is not None:
        if sum_out is None:
            sum_out = new(x)
        else:
            if sum_out.shape != x.shape or sum_out.dtype is not dtype or sum_out.get_device() != index:
                raise ValueError(f"sum_out must be {tuple(x.shape)} {dtype} on {device}")
            s_stride = _row_layout(sum_out, K)
            if not s_stride:
                raise ValueError("sum_out must consist of packed rows evenly apart")
            _check_sum(sum_out, s_stride, x, K, "x")
            _check_sum(sum_out, s_stride, residual, K, "residual")
        r_stride = _row_layout(residual, K)
        if not r_stride:
            residual, r_stride = residual.contiguous(), K
    out = data = codes = scales = None
    apart = 0
    if not quantize or keep_rows:
        out = new(x)
    if quantize:
        apart = (M + 255) // 256 * 256
        data = torch.empty(QuantizedRows.nbytes(M, K), dtype=torch.uint8, device=device)
        codes = data.data_ptr()
        scales = codes + (K + 127) // 128 * 128 * M
    if given:  # (a graph that saved it has to see this)
        increment_version(sum_out)
    _lib.call_on(device, "gdn_rms_norm", x.data_ptr(), x_stride, _lib.ptr(residual), r_stride, _lib.ptr(sum_out), s_stride,
                 _lib.ptr(weight), float(eps), _lib.dtype_code(dtype), _lib.ptr(out), codes, scales, apart, M, K,
                 _stream(device))
    normed = out if not quantize else QuantizedRows._made(x.shape, dtype, data, out)
    return normed if residual is None else (normed, sum_out)


def _check_sum(out: torch.Tensor, stride: int, src: torch.Tensor, K: int, name: str) -> None:
    """``out``, rows of K ``stride`` apart, is ``src`` itself (of one row the stride says
    nothing) or does not overlap it."""

    apart = _row_layout(src, K)
    if out.data_ptr() == src.data_ptr() and apart == stride:
        return
    if apart == stride and not rows_overlap(out.data_ptr(), src.data_ptr(), stride, K, K, out.numel() // K,
                                                          out.element_size()):
        return
    ends = [(t.data_ptr(), t.data_ptr() + (sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1) * t.element_size())
            for t in (out, src) if t.numel()]
    if len(ends) == 2 and ends[0][0] < ends[1][1] and ends[1][0] < ends[0][1]:
        raise ValueError(f"sum_out must be {name} itself or not overlap it")
