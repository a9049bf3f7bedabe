"""Embedding lookup with scaling, and its gradient by sorted tokens.

The first step of a packed forward pass (the token embeddings that
``models/lfm2_5/encoder.py:202-240`` looks up) with the gradient of its table.
"""

from __future__ import annotations

import math

import torch

from .. import _lib
from ..ops import _raw_stream, dtype_code, even_rows, launch, refuse_tangents, require_device


def _launch(ids, table, scale, padding):
    v, d = table.shape
    out = torch.empty((*ids.shape, d), dtype=table.dtype, device=table.device)
    if ids.numel():
        launch(table.device, _lib.LIB.mf_embed, ids.data_ptr(), ids.element_size(),
               table.data_ptr(), even_rows(table)[1], dtype_code(table), ids.numel(), v, d,
               padding, scale, out.data_ptr(), _raw_stream(table.device.index))
    return out


def _launch_gradient(dout, ids, v, scale, padding):
    n, d, device = ids.numel(), dout.shape[-1], dout.device
    if not n:
        return dout.new_zeros((v, d))
    dout, step = even_rows(dout)
    dtable = torch.empty((v, d), dtype=dout.dtype, device=device)
    ws_bytes = _lib.LIB.mf_embed_bwd_workspace_bytes(n, v, d)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    launch(device, _lib.LIB.mf_embed_bwd, ids.data_ptr(), ids.element_size(), dout.data_ptr(),
           step, dtype_code(dout), n, v, d, padding, scale, dtable.data_ptr(), ws.data_ptr(),
           ws_bytes, _raw_stream(device.index))
    return dtable


class Embed(torch.autograd.Function):
    """The lookup with a HIP forward and a HIP backward; the gradient reaches the table.  It is
    linear in what comes in, and the lookup is its transpose: differentiable as often as asked."""

    @staticmethod
    def forward(ctx, ids, table, scale, padding):
        ctx.save_for_backward(ids)
        ctx.args = (table.shape[0], scale, padding)
        return _launch(ids, table, scale, padding)

    @staticmethod
    def backward(ctx, dout):
        gradient = EmbedGradient.apply if torch.is_grad_enabled() else _launch_gradient
        return None, gradient(dout, ctx.saved_tensors[0], *ctx.args), None, None


class EmbedGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, dout, ids, v, scale, padding):
        ctx.save_for_backward(ids)
        ctx.args = (scale, padding)
        return _launch_gradient(dout, ids, v, scale, padding)

    @staticmethod
    def backward(ctx, g):
        lookup = Embed.apply if torch.is_grad_enabled() else _launch
        return lookup(ctx.saved_tensors[0], even_rows(g)[0], *ctx.args), None, None, None, None


def embed(ids: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0,
          padding_id: int | None = None) -> torch.Tensor:
    """``scale * table[ids]``: ids of any shape, ``table [V, D]``, the result ``[*ids, D]``.

    Ids outside ``0 .. V-1`` and ``padding_id`` have rows of zeros and no part in the
    gradient (nothing is read back to the host to refuse them).  The table's gradient
    is dense, in the table's dtype; a row's tokens are added in float32 in an order that
    depends on the ids alone, so the same inputs give the same bits.  Differentiable
    in the table.
    """
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
    ids, table = ids.contiguous(), even_rows(table)[0]
    if table.requires_grad and torch.is_grad_enabled():
        return Embed.apply(ids, table, scale, padding_id)
    return _launch(ids, table, scale, padding_id)
