"""Layer norm and RMS norm over the hidden width, with their backward passes.

The norms of ``kernels/normalization.py:7-22`` (``rms_norm``) and of the layer norm
of ``kernels/bidirectional.py`` over the last dimension, whatever its width.
float32 arithmetic, each output rounded once; the per-head norm of
:func:`prologue.qk_norm_rope` rounds the normalised value before the gain, as the
reference's declared types do, so results differ in the last bit.
"""

from __future__ import annotations

import math

import torch

from .. import _lib
from ..ops import (_ptr, _raw_stream, dtype_code, even_rows, launch, refuse_second_order,
                   refuse_tangents, require_device)


def _launch(x, weight, bias, eps, center, with_stats):
    d = x.shape[-1]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    rows = x.numel() // d
    stats = torch.empty(2 * rows, dtype=torch.float32, device=x.device) if with_stats else None
    if rows:
        launch(x.device, _lib.LIB.mf_norm, x.data_ptr(), even_rows(x)[1], weight.data_ptr(),
               _ptr(bias), dtype_code(x), dtype_code(weight), rows, d, center, eps, y.data_ptr(),
               _ptr(stats), _raw_stream(x.device.index))
    return y, stats


class Norm(torch.autograd.Function):
    """A norm with a HIP forward and a HIP backward; gradients reach x, weight and bias."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, center):
        y, stats = _launch(x, weight, bias, eps, center, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.center = center
        return y

    @staticmethod
    def backward(ctx, dy):
        refuse_second_order("the norm")
        x, weight, stats = ctx.saved_tensors
        d, device = x.shape[-1], x.device
        rows = x.numel() // d
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        if not rows:
            zeros = torch.zeros_like
            return (zeros(x) if need_x else None, zeros(weight) if need_w else None,
                    zeros(weight) if need_b else None, None, None)
        dx = torch.empty(x.shape, dtype=x.dtype, device=device) if need_x else None
        dw = torch.empty(d, dtype=weight.dtype, device=device) if need_w else None
        db = torch.empty(d, dtype=weight.dtype, device=device) if need_b else None
        code = dtype_code(x)
        ws, ws_bytes = None, 0
        if need_w or need_b:
            ws_bytes = _lib.LIB.mf_norm_bwd_workspace_bytes(rows, d, code)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
        dy, dy_step = even_rows(dy)
        launch(device, _lib.LIB.mf_norm_bwd, x.data_ptr(), even_rows(x)[1], weight.data_ptr(),
               stats.data_ptr(), dy.data_ptr(), dy_step, code, dtype_code(weight), rows, d,
               ctx.center, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), ws_bytes,
               _raw_stream(device.index))
        return dx, dw, db, None, None


def _norm(what, x, weight, bias, eps, center):
    d = x.shape[-1] if x.dim() else 0
    if not d:
        raise ValueError("x must be [..., D] with D positive")
    dtype_code(x)
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != (d,):
            raise ValueError(f"{name} must be [{d}], got {list(p.shape)}")
        if p.dtype is not x.dtype and p.dtype is not torch.float32:
            raise ValueError(f"{name} must be {x.dtype} or float32 (got {p.dtype})")
    if bias is not None and bias.dtype is not weight.dtype:
        raise ValueError(f"weight and bias must share one dtype (got {weight.dtype} and {bias.dtype})")
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative (got {eps})")
    refuse_tangents(what, x, weight, bias)
    if bias is None:
        require_device(x, weight)
    else:
        require_device(x, weight, bias)
        bias = bias.contiguous()
    weight = weight.contiguous()
    x = even_rows(x)[0]
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (bias is not None and bias.requires_grad)):
        return Norm.apply(x, weight, bias, eps, center)
    return _launch(x, weight, bias, eps, center, False)[0]


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of ``x [..., D]``.

    ``weight [D]`` and ``bias [D]`` are in x's dtype or, both, in float32; their
    gradients have their dtype.  Mean and spread are those of the row itself, in
    float32.  D up to 16384, up to 2**22 rows, evenly spaced or copied.
    Differentiable in x, weight and bias, once; the same inputs give the same bits.
    """
    return _norm("layer_norm", x, weight, bias, eps, True)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-5) -> torch.Tensor:
    """``x / sqrt(mean(x * x) + eps) * weight`` over the last dimension; as :func:`layer_norm`."""
    return _norm("rms_norm", x, weight, None, eps, False)
