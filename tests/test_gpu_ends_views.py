"""Operands that are views of a negation: torch keeps the sign beside the memory."""

import pytest
import torch

from mfattn.kernels import distillation, embedding, normalization

pytestmark = pytest.mark.gpu


def _negated(t):
    """``t`` over memory that holds ``-t``."""
    view = torch._neg_view((-t.detach()).clone())
    assert view.is_neg()
    return view


def _imaginary(t):
    """``t``, as the imaginary parts of a conjugate: every second value of its memory, negated."""
    view = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert view.is_neg()
    return view


@pytest.mark.parametrize("negated", [_negated, _imaginary])
@pytest.mark.parametrize("d", [1, 40])
def test_norms(d, negated, device):
    x, w, b, dy = (torch.randn(s, device=device) for s in ((6, d), (d,), (d,), (6, d)))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = normalization.layer_norm(*leaves)
    want = torch.autograd.grad(y, leaves, dy)
    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            assert torch.equal(normalization.layer_norm(negated(x), negated(w), negated(b)), y)
            assert torch.equal(normalization.layer_norm(*leaves[:2], negated(b)), y)
    moved = [negated(t).requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(normalization.layer_norm(*moved), moved, negated(dy))
    for p, q in zip(got, want):
        assert torch.equal(p, q)


@pytest.mark.parametrize("negated", [_negated, _imaginary])
@pytest.mark.parametrize("d", [1, 40])
def test_embedding(d, negated, device):
    ids = torch.tensor([3, 0, 3, 7], device=device)
    table, dout = torch.randn(9, d, device=device), torch.randn(4, d, device=device)
    leaf = table.clone().requires_grad_()
    out = embedding.embed(ids, leaf, scale=2.0)
    (want,) = torch.autograd.grad(out, leaf, dout)
    assert torch.equal(embedding.embed(ids, negated(table), scale=2.0), out)
    moved = negated(table).requires_grad_()
    (got,) = torch.autograd.grad(embedding.embed(ids, moved, scale=2.0), moved, negated(dout))
    assert torch.equal(got, want)


@pytest.mark.parametrize("negated", [_negated, _imaginary])
@pytest.mark.parametrize("v, k", [(50, 4), (1, 1)])
def test_distillation(v, k, negated, device):
    z, t, total, weights = (torch.randn(s, device=device) for s in ((5, v), (5, k), (5,), (5,)))
    total = total + 4
    ids = torch.rand(5, v, device=device).argsort(1)[:, :k].contiguous()
    more = {"teacher_total": total, "weights": weights}
    loss, grad = distillation.top_logits_loss_and_gradient(z, t, ids, **more)
    odd = {name: negated(x) for name, x in more.items()}
    for how in (odd, more):
        got = distillation.top_logits_loss_and_gradient(negated(z), negated(t), ids, **how)
        assert torch.equal(got[0], loss) and torch.equal(got[1], grad)
    got = distillation.top_logits_loss_and_gradient(z, negated(t), ids, **odd, out=torch.empty_like(z))
    assert torch.equal(got[0], loss) and torch.equal(got[1], grad)
    up = torch.randn(5, device=device)
    leaf = z.clone().requires_grad_()
    (want,) = torch.autograd.grad(distillation.top_logits_loss(leaf, t, ids, **more), leaf, up)
    moved = negated(z).requires_grad_()
    (got,) = torch.autograd.grad(distillation.top_logits_loss(moved, negated(t), ids, **odd), moved,
                                 negated(up))
    assert torch.equal(got, want)
    with pytest.raises(ValueError, match="out must"):
        distillation.top_logits_loss_and_gradient(z, t, ids, out=_negated(z), **more)
