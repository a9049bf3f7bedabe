"""Forward-mode derivatives of the rotary embedding, and the calls that have none."""

import pytest
import torch
from torch.autograd import forward_ad

from _paged import close, turned
from mfattn.kernels import paged, rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tangents_turn_with_their_tensors(dtype, device):
    rot = rotary.Rotary(64, rotary_dim=32, interleaved=True, scaling="linear", factor=2.0)
    g = torch.Generator(device=device).manual_seed(1)
    q, tq = (torch.randn(2, 9, 4, 64, generator=g, device=device).to(dtype) for _ in range(2))
    k, tk = (torch.randn(2, 9, 2, 64, generator=g, device=device).to(dtype) for _ in range(2))
    pos = torch.arange(18, device=device, dtype=torch.int32).view(2, 9) * 100
    plain = rotary.rotate(q, k, rot, pos)
    with forward_ad.dual_level():
        qo, ko = rotary.rotate(forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk), rot, pos)
        (qo, dq), (ko, dk) = forward_ad.unpack_dual(qo), forward_ad.unpack_dual(ko)
        assert torch.equal(qo, plain[0]) and torch.equal(ko, plain[1])
        assert dq is not None and dk is not None
        close(dq, *turned(tq, pos, rot), "query's tangent")
        close(dk, *turned(tk, pos, rot), "key's tangent")
        # one of two, without gradients, and no key
        with torch.no_grad():
            qo, ko = rotary.rotate(q, forward_ad.make_dual(k, tk), rot, pos)
        assert torch.equal(forward_ad.unpack_dual(ko).tangent, dk)
        one = forward_ad.unpack_dual(qo).tangent
        assert one is None or not one.any()
        alone, none = rotary.rotate(forward_ad.make_dual(q, tq), None, rot, pos)
        assert none is None and torch.equal(forward_ad.unpack_dual(alone).tangent, dq)
        # a tensor that takes part in both modes
        both = forward_ad.make_dual(q.clone().requires_grad_(), tq)
        out, _ = rotary.rotate(both, None, rot, pos)
        assert torch.equal(forward_ad.unpack_dual(out).tangent, dq)
        # forward over reverse: the tangent of a gradient is that of what comes in
        x = q.clone().requires_grad_()
        out, _ = rotary.rotate(x, None, rot, pos)
        (grad,) = torch.autograd.grad(out, x, forward_ad.make_dual(q, tq))
        close(forward_ad.unpack_dual(grad).tangent, *turned(tq, pos, rot, back=True), "over reverse")
        # nothing dual: as without
        qo, ko = rotary.rotate(q, k, rot, pos)
        assert torch.equal(qo, plain[0]) and forward_ad.unpack_dual(qo).tangent is None


def test_a_tangent_has_a_gradient(device):
    """Reverse over forward: the tangent is a rotation of its own, so its gradient turns back."""
    rot = rotary.Rotary(64)
    g = torch.Generator(device=device).manual_seed(3)
    q, t, w = (torch.randn(1, 7, 3, 64, generator=g, device=device) for _ in range(3))
    t.requires_grad_()
    with forward_ad.dual_level():
        out, _ = rotary.rotate(forward_ad.make_dual(q, t), None, rot)
        (grad,) = torch.autograd.grad(forward_ad.unpack_dual(out).tangent, t, w)
    close(grad, *turned(w, torch.arange(7)[None], rot, back=True), "reverse over forward")


def test_paged_calls_take_no_tangent(device):
    kp, vp = (torch.zeros(4, 16, 2, 64, device=device) for _ in range(2))
    starts = torch.tensor([0, 3], dtype=torch.int32, device=device)
    plan = paged.plan(starts, starts[1:], torch.zeros(1, 1, dtype=torch.int32, device=device), kp,
                      tokens=3, query_heads=4)
    q, k = torch.ones(3, 4, 64, device=device), torch.ones(3, 2, 64, device=device)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(k, torch.ones_like(k))
        with pytest.raises(ValueError, match="tangent"):
            paged.append(dual, k, kp, vp, plan)
        with pytest.raises(ValueError, match="tangent"):
            paged.append(k, k, kp, vp, plan, key_gain=forward_ad.make_dual(k[0, 0], k[0, 0]))
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
            paged.attention(forward_ad.make_dual(q, q), kp, vp, plan)
        paged.append(k, k, kp, vp, plan)
        assert torch.isfinite(paged.attention(q, kp, vp, plan)).all()
