"""Embedding lookup with scaling, and its gradient by sorted tokens.

The first step of a packed forward pass (the token embeddings that
``models/lfm2_5/encoder.py:202-240`` looks up) with the gradient of its table.
"""

from __future__ import annotations

import math

import torch

from .. import _nodes
from .._nodes import even_rows
from ..ops import dtype_code, refuse_tangents, require_device


def embed(ids: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0,
          padding_id: int | None = None) -> torch.Tensor:
    """``scale * table[ids]``: ids of any shape, ``table [V, D]``, the result ``[*ids, D]``.

    Ids outside ``0 .. V-1`` and ``padding_id`` have rows of zeros and no part in the
    gradient (nothing is read back to the host to refuse them).  The table's gradient
    is dense, in the table's dtype; a row's tokens are added in float32 in an order that
    depends on the ids alone, so the same inputs give the same bits.  V up to 2**27, D up
    to 65536, up to 2**24 ids and 2**34 values.  Differentiable in the table.  (A
    backward captured into a graph: see :func:`normalization.layer_norm`.)
    """
    out = _nodes.usual_embed(ids, table, scale, padding_id)
    return _other(ids, table, scale, padding_id) if out is None else out


def _other(ids, table, scale, padding_id):
    """A call whose operands are not all of the ordinary kind, or wrong."""
    if table.dim() != 2 or not table.shape[0] or not table.shape[1]:
        raise ValueError("table must be [V, D] with V and D positive")
    if ids.is_floating_point() or ids.is_complex() or ids.dtype is torch.bool:
        raise ValueError(f"ids must be integers, got {ids.dtype}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite (got {scale})")
    if padding_id is None:
        padding_id = -1
    elif not -2 ** 63 <= padding_id < 2 ** 63:
        raise ValueError(f"padding_id must be a 64-bit integer (got {padding_id})")
    dtype_code(table)
    refuse_tangents("embed", table)
    require_device(table, ids)
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        ids = ids.to(torch.int64)
    return _nodes.embed(ids.resolve_neg().contiguous(), even_rows(table), scale, padding_id,
                        table.requires_grad and torch.is_grad_enabled())
