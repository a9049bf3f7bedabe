"""Rotary position embeddings: half and interleaved layouts, part of the head, long contexts.

The general form of ``apply_rotary`` (``kernels/rotary.py:7-39`` of the
reference, which rotates whole heads in the half layout): pair ``i`` of the
``rotary_dim`` rotated dims turns by ``position * frequencies[i]`` and the
other dims pass.  Arithmetic is float32 (turns are counted in whole
numbers, so no error grows with the position), rounded once to the tensors'
dtype; :func:`prologue.qk_norm_rope` rounds every step, as the reference's
declared types do, so its results differ in the last bit.
"""

from __future__ import annotations

import ctypes
import math

import torch

from .. import _lib
from ..ops import _ptr, _raw_stream, carries_tangent, dtype_code, launch, require_device, token_rows
from .prologue import _positions

_SCALINGS = ("none", "linear", "base", "bands", "ramp")


class Rotary:
    """The frequencies of a rotary embedding, made once from a model's configuration.

    ``head_dim`` is the width of a head, of which the first ``rotary_dim``
    (default: all) rotate; ``interleaved`` pairs dims ``(2i, 2i + 1)`` instead
    of ``(i, i + rotary_dim / 2)``.  ``frequencies[i] = theta ** (-2i /
    rotary_dim)`` radians per position, stretched for contexts ``factor`` times
    longer than the model was trained on by ``scaling``:

    * ``none``
    * ``linear``: every frequency divided by ``factor``;
    * ``base``: ``theta`` multiplied by ``factor ** (rotary_dim / (rotary_dim - 2))``,
      which keeps the first frequency and divides the last by ``factor``;
    * ``bands``: by the turns a pair makes in ``original_length`` positions: kept
      above ``fast`` (default 4), divided by ``factor`` below ``slow`` (default 1),
      blended linearly in the turns between;
    * ``ramp``: by the pair's index: kept up to the index whose pair makes ``fast``
      (default 32) turns in ``original_length``, divided by ``factor`` from the one
      with ``slow`` (default 1) on, blended linearly in the index between; the
      rotated dims are also multiplied by ``magnitude`` (default ``0.1 ln(factor) + 1``).

    Given ``frequencies`` (``rotary_dim / 2`` numbers) replace all of this.
    """

    def __init__(self, head_dim: int, *, theta: float = 10000.0, rotary_dim: int | None = None,
                 interleaved: bool = False, scaling: str | None = None, factor: float = 1.0,
                 original_length: int | None = None, fast: float | None = None,
                 slow: float = 1.0, magnitude: float | None = None, frequencies=None):
        r = head_dim if rotary_dim is None else rotary_dim
        scaling = "none" if scaling is None else scaling
        if head_dim < 2 or head_dim % 2 or head_dim > _lib.ROTATE_MAX_HEAD_DIM:
            raise ValueError(f"head_dim must be even and in [2, {_lib.ROTATE_MAX_HEAD_DIM}] "
                             f"(got {head_dim})")
        if r < 2 or r % 2 or r > min(head_dim, _lib.ROTATE_MAX_DIM):
            raise ValueError(f"rotary_dim must be even and in [2, min(head_dim, "
                             f"{_lib.ROTATE_MAX_DIM})] (got {r} of {head_dim})")
        if scaling not in _SCALINGS:
            raise ValueError(f"Unsupported rotary scaling: {scaling}")
        if not (theta > 1 and math.isfinite(theta)):
            raise ValueError("theta must be finite and above 1")
        if not (factor >= 1 and math.isfinite(factor)):
            raise ValueError("factor must be finite and at least 1")
        if scaling in ("bands", "ramp"):
            fast = (4.0 if scaling == "bands" else 32.0) if fast is None else fast
            if not original_length or original_length < 1:
                raise ValueError(f"{scaling} scaling needs original_length")
            if not 0 < slow < fast:
                raise ValueError("scaling needs 0 < slow < fast turns")
        if frequencies is not None:
            freqs = [float(f) for f in frequencies]
            if len(freqs) != r // 2:
                raise ValueError(f"frequencies must hold rotary_dim / 2 = {r // 2} numbers")
        else:
            freqs = _scaled(r, theta, scaling, factor, original_length, fast, slow)
        if magnitude is None:
            magnitude = 1.0 + 0.1 * math.log(factor) if scaling == "ramp" else 1.0
        if not all(math.isfinite(f) for f in (*freqs, magnitude)):
            raise ValueError("frequencies and magnitude must be finite")
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, r, bool(interleaved)
        self.frequencies, self.magnitude = tuple(freqs), float(magnitude)
        self._turns = (ctypes.c_uint64 * len(freqs))()
        _lib.check(_lib.LIB.mf_rotary_turns((ctypes.c_double * len(freqs))(*freqs), len(freqs),
                                            self._turns))
        # the C ABI's arguments: host array, rotary_dim, interleaved, magnitude
        self._args = (ctypes.addressof(self._turns), r, int(self.interleaved), self.magnitude)

    def __reduce__(self):
        # (copies and pickles make turns of their own: the arguments hold an address)
        return _rotary_of, (self.head_dim, self.rotary_dim, self.interleaved, self.frequencies,
                            self.magnitude)

    def __repr__(self) -> str:
        return (f"Rotary(head_dim={self.head_dim}, rotary_dim={self.rotary_dim}, "
                f"interleaved={self.interleaved}, magnitude={self.magnitude:g})")


def _rotary_of(head_dim, rotary_dim, interleaved, frequencies, magnitude) -> Rotary:
    return Rotary(head_dim, rotary_dim=rotary_dim, interleaved=interleaved,
                  frequencies=frequencies, magnitude=magnitude)


def _scaled(r, theta, scaling, factor, length, fast, slow) -> list[float]:
    if scaling == "base":
        # of a single pair there is no last frequency to slow
        theta = theta * factor ** (r / (r - 2)) if r > 2 else theta
    freqs = [theta ** (-2 * i / r) for i in range(r // 2)]
    if scaling == "linear":
        return [f / factor for f in freqs]
    if scaling == "bands":
        keep = [(length * f / (2 * math.pi) - slow) / (fast - slow) for f in freqs]
        keep = [min(max(x, 0.0), 1.0) for x in keep]
        return [f * (x + (1 - x) / factor) for f, x in zip(freqs, keep)]
    if scaling == "ramp":
        # index whose pair makes n turns in `length` positions
        lo, hi = (r * math.log(length / (2 * math.pi * n)) / (2 * math.log(theta))
                  for n in (fast, slow))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), r - 1)
        drop = [min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0) for i in range(r // 2)]
        return [f * (1 - x + x / factor) for f, x in zip(freqs, drop)]
    return freqs


def _launch(q, k, positions, rotary, backward):
    """Rotates q and k ([B, T, H, D] or [N, H, D], either None) into new dense tensors."""
    one = q if q is not None else k
    shape, dtype, device = one.shape, one.dtype, one.device
    tokens, seq_len = (shape[0] * shape[1], shape[1]) if len(shape) == 4 else (shape[0], shape[0])
    qp = kp = qo = ko = q_out = k_out = None
    hq = hkv = q_stride = k_stride = 0
    if q is not None:
        q, q_stride = token_rows(q)
        q_out = torch.empty(q.shape, dtype=dtype, device=device)
        hq, qp, qo = q.shape[-2], q.data_ptr(), q_out.data_ptr()
    if k is not None:
        k, k_stride = token_rows(k)
        k_out = torch.empty(k.shape, dtype=dtype, device=device)
        hkv, kp, ko = k.shape[-2], k.data_ptr(), k_out.data_ptr()
    turns, rotary_dim, interleaved, magnitude = rotary._args
    launch(device, _lib.LIB.mf_rotate, qp, q_stride, kp, k_stride, _ptr(positions), turns,
           dtype_code(one), tokens, seq_len, hq, hkv, rotary.head_dim, rotary_dim, interleaved,
           magnitude, backward, qo, ko, _raw_stream(device.index))
    return q_out, k_out


class Rotate(torch.autograd.Function):
    """Rotation of queries and keys in one launch; the backward turns the gradients back,
    which is a rotation again (and differentiable as one), and tangents turn as their
    tensors do."""

    @staticmethod
    def forward(ctx, q, k, positions, rotary, back):
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        ctx.rotary, ctx.back = rotary, back
        ctx.shapes = tuple(None if x is None else x.shape for x in (q, k))
        ctx.set_materialize_grads(False)
        return _launch(q, k, positions, rotary, back)

    @staticmethod
    def backward(ctx, dq, dk):
        dq = dq if ctx.needs_input_grad[0] else None
        dk = dk if ctx.needs_input_grad[1] else None
        if dq is None and dk is None:
            return None, None, None, None, None
        turn = Rotate.apply if torch.is_grad_enabled() or carries_tangent(dq, dk) else _launch
        dq, dk = turn(dq, dk, ctx.saved_tensors[0], ctx.rotary, not ctx.back)
        return dq, dk, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        turn = Rotate.apply if torch.is_grad_enabled() else _launch
        out = turn(tq, tk, ctx.saved_tensors[0], ctx.rotary, ctx.back)
        one = out[0] if out[1] is None else out[1]
        # (an output that has a tangent beside it needs one too)
        return tuple(one.new_zeros(s) if t is None and s is not None else t
                     for t, s in zip(out, ctx.shapes))


def rotate(query: torch.Tensor, key: torch.Tensor | None, rotary: Rotary, positions=None
           ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotate ``query [B, T, Hq, D]`` and ``key [B, T, Hkv, D]`` (or ``[N, H, D]`` both).

    ``positions`` are integers: a scalar, ``[T]`` or ``[B, T]`` (``[N]`` for
    three dimensions) in int32's range; ``None`` means ``0 .. T-1`` on every row.
    ``key`` may be ``None``.  Slices of one projection are read where they are as
    long as each head is dense and tokens are evenly spaced.  Differentiable in
    both, in reverse and in forward mode.  A backward is captured into a graph
    together with its forward and while no eager graph of the same leaves is
    alive, as for any operation: autograd accumulates a leaf's
    gradient on the stream of its oldest graph.
    """
    if not isinstance(rotary, Rotary):
        raise ValueError("rotary must be a Rotary")
    if query.dim() not in (3, 4):
        raise ValueError("query must be [B, T, H, D] or [N, H, D]")
    if query.shape[-1] != rotary.head_dim:
        raise ValueError(f"the rotary embedding is for heads of {rotary.head_dim}, "
                         f"the query has {query.shape[-1]}")
    if key is not None and (key.shape[:-2] != query.shape[:-2] or key.shape[-1] != query.shape[-1]
                            or key.dtype != query.dtype):
        raise ValueError("query and key must share batch, length, head_dim and dtype")
    dtype_code(query)
    if positions is not None:
        positions = torch.as_tensor(positions)
        if (positions.is_floating_point() or positions.is_complex()
                or positions.dtype is torch.bool):
            raise ValueError(f"positions must be integers, got {positions.dtype}")
    device = require_device(query) if key is None else require_device(query, key)
    if query.dim() == 4:
        pos = _positions(positions, query.shape[0], query.shape[1], device)
    else:
        pos = _positions(positions, 1, query.shape[0], device)
    if (not torch.is_grad_enabled() or not (query.requires_grad
                                            or (key is not None and key.requires_grad))) \
            and not carries_tangent(query, key):
        return _launch(query, key, pos, rotary, False)
    return Rotate.apply(query, key, pos, rotary, False)
