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

from .. import _nodes
from .._nodes import even_rows
from ..ops import dtype_code, refuse_tangents, require_device


def _norm(what, x, weight, bias, eps, center):
    y = _nodes.usual_norm(x, weight, bias, eps, center)
    return _other(what, x, weight, bias, eps, center) if y is None else y


def _other(what, x, weight, bias, eps, center):
    """A call whose operands are not all of the ordinary kind, or wrong."""
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
        bias = bias.resolve_neg().contiguous()
    record = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                          or (bias is not None and bias.requires_grad))
    return _nodes.norm(even_rows(x), weight.resolve_neg().contiguous(), bias, eps, center, record)


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of ``x [..., D]``.

    ``weight [D]`` and ``bias [D]`` are in x's dtype or, both, in float32; their
    gradients have their dtype.  Mean and spread are those of the row itself, in
    float32.  D up to 16384, up to 2**22 rows, evenly spaced or copied.
    Differentiable in x, weight and bias, once; the same inputs give the same bits.
    A backward is captured into a graph together with its forward and while no eager
    graph of the same leaves is alive, as for any operation: autograd accumulates a
    leaf's gradient on the stream of its oldest graph.
    """
    return _norm("layer_norm", x, weight, bias, eps, True)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-5) -> torch.Tensor:
    """``x / sqrt(mean(x * x) + eps) * weight`` over the last dimension; as :func:`layer_norm`."""
    return _norm("rms_norm", x, weight, None, eps, False)
