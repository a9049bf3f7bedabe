"""Distillation from a teacher's top logits: the loss over the vocabulary and its gradient.

The last step of a packed training pass (beside the causal and pointer losses of the
reference's ``objectives/``), for a teacher of which only the largest logits of
every token are kept.  With ``q = softmax(logits / temperature)`` and the teacher's
masses ``p`` over its entries::

    loss = weight * temperature ** 2 * (sum_k p_k (log p_k - log q_k) + r (log r - log s))

``p`` is the softmax of the entries, and ``r`` zero; or, where ``teacher_total`` (the
logarithm of the sum of the teacher's exponentials over its whole vocabulary, at
this temperature) is given, ``exp(teacher / temperature - teacher_total)``, ``r`` what
they leave of one, and ``s`` what the student has on the ids without an entry.
"""

from __future__ import annotations

import torch

from .. import _nodes
from .._nodes import even_rows
from ..ops import dtype_code, refuse_tangents, require_device


def _checked(what, logits, teacher, ids, total, weights, temperature):
    lead = logits.shape[:-1]
    if not logits.dim() or not logits.shape[-1]:
        raise ValueError("logits must be [..., V] with V positive")
    if ids.shape[:-1] != lead or ids.dim() != logits.dim() or not ids.shape[-1] \
            or teacher.shape != ids.shape:
        raise ValueError(f"teacher_logits and teacher_ids must be {[*lead, 'K']}, got "
                         f"{list(teacher.shape)} and {list(ids.shape)}")
    if ids.is_floating_point() or ids.is_complex() or ids.dtype is torch.bool:
        raise ValueError(f"teacher_ids must be integers, got {ids.dtype}")
    dtype_code(logits)
    dtype_code(teacher)
    tensors = [logits, teacher, ids]
    for name, t in (("teacher_total", total), ("weights", weights)):
        if t is None:
            continue
        if t.shape != lead:
            raise ValueError(f"{name} must be {list(lead)}, got {list(t.shape)}")
        if not t.is_floating_point():
            raise ValueError(f"{name} must be floating, got {t.dtype}")
        tensors.append(t)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"temperature must be in [1e-6, 1e6] (got {temperature})")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (teacher, total, weights)):
        raise ValueError(f"{what} has a gradient for the logits alone; detach the teacher and "
                         "the weights")
    refuse_tangents(what, logits, teacher, total, weights)
    require_device(*tensors)
    if ids.dtype is not torch.int32 and ids.dtype is not torch.int64:
        ids = ids.to(torch.int64)

    def dense(t):
        return t.detach().resolve_neg().contiguous()

    def row(t):
        return None if t is None else dense(t.to(torch.float32))

    return dense(teacher), dense(ids), row(total), row(weights)


def top_logits_loss(logits: torch.Tensor, teacher_logits: torch.Tensor,
                    teacher_ids: torch.Tensor, *, temperature: float = 1.0,
                    teacher_total: torch.Tensor | None = None,
                    weights: torch.Tensor | None = None) -> torch.Tensor:
    """The loss of every row (float32, ``logits.shape[:-1]``) against a teacher's top logits.

    ``logits [..., V]`` are the student's; ``teacher_logits`` and ``teacher_ids [..., K]``
    the teacher's entries, in any order.  An entry whose id is outside ``0 .. V-1`` (-1,
    say) is not there; entries with the same id add up.  ``teacher_total [...]``
    counts the teacher's other tokens in (see the module).  ``weights [...]`` multiplies
    the losses; a row of weight zero has loss and gradient zero whatever its logits
    hold, and so has a row without entries (where no total is given).  V up to
    393216, K up to 1024, temperatures in [1e-6, 1e6].  The teacher's masses and the
    logarithms are 64-bit, exponentials of logits and their sums float32: a loss is
    off by some 1e-7 times ``weight * temperature ** 2``.  With a total this holds however far the
    student's logits of the entries are above all others; the loss is infinite only where an
    entry with mass, or every id without one while ``r`` is positive, has the logit -infinity.
    Differentiable in the logits, once;
    :func:`top_logits_loss_and_gradient` needs half the memory and two passes over the
    logits instead of three.  (A backward captured into a graph: see
    :func:`normalization.layer_norm`.)
    """
    loss = _nodes.usual_distill(logits, teacher_logits, teacher_ids, teacher_total, weights, temperature,
                                False)
    if loss is not None:
        return loss
    teacher, ids, total, weights = _checked("top_logits_loss", logits, teacher_logits, teacher_ids,
                                            teacher_total, weights, temperature)
    record = logits.requires_grad and torch.is_grad_enabled()
    return _nodes.distill(even_rows(logits), teacher, ids, total, weights, temperature, record, None)


def top_logits_loss_and_gradient(logits: torch.Tensor, teacher_logits: torch.Tensor,
                                 teacher_ids: torch.Tensor, *, temperature: float = 1.0,
                                 teacher_total: torch.Tensor | None = None,
                                 weights: torch.Tensor | None = None,
                                 out: torch.Tensor | None = None
                                 ) -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`top_logits_loss` and the gradient of the losses' sum, in one pass over the logits.

    What the sum of losses is to be multiplied by (one over the tokens, say) goes into
    ``weights``; the gradient then goes straight into the projection's backward pass.  It is
    written to ``out``, in the logits' dtype, which may be the logits themselves.  No
    graph is recorded: logits that require a gradient are refused unless under
    ``torch.no_grad()``.
    """
    if out is None:
        both = _nodes.usual_distill(logits, teacher_logits, teacher_ids, teacher_total, weights,
                                    temperature, True)
        if both is not None:
            return both
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("top_logits_loss_and_gradient records no graph; call it under "
                         "torch.no_grad(), or top_logits_loss")
    teacher, ids, total, weights = _checked("top_logits_loss_and_gradient", logits, teacher_logits,
                                            teacher_ids, teacher_total, weights, temperature)
    if out is None:
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        return _nodes.distill(even_rows(logits), teacher, ids, total, weights, temperature, False,
                              grad), grad
    if out.shape != logits.shape or out.dtype is not logits.dtype or out.device != logits.device:
        raise ValueError(f"out must be a {logits.dtype} {list(logits.shape)} on {logits.device}")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out must not require a gradient")
    if even_rows(out) is not out:
        raise ValueError("out must have evenly spaced rows and a dense last dimension")
    same = out.data_ptr() == logits.data_ptr() and out.stride() == logits.stride()
    memory = out.untyped_storage().data_ptr() or None  # (none of an empty tensor)
    if not same and memory == logits.untyped_storage().data_ptr():
        raise ValueError("out must be the logits or share no memory with them")
    # (rows are written while others' entries are yet to be read)
    if any(t is not None and memory == t.untyped_storage().data_ptr()
           for t in (teacher, ids, total, weights)):
        raise ValueError("out must share no memory with the teacher or the weights")
    loss = _nodes.distill(even_rows(logits), teacher, ids, total, weights, temperature, False, out)
    torch.autograd.graph.increment_version(out)
    return loss, out
