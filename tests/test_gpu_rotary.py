"""Rotary embeddings against their definition in float64: layouts, widths, positions, gradients."""

import numpy as np
import pytest
import torch

from _helpers import say
from _paged import close, turned
from mfattn.kernels import rotary

pytestmark = pytest.mark.gpu


def _qk(dtype, shape, hq, hkv, d, device, seed=0):
    """q and k as parts of one projection (with values behind them)."""
    g = torch.Generator(device=device).manual_seed(seed)
    fused = torch.randn(*shape, (hq + 2 * hkv) * d, generator=g, device=device).to(dtype)
    return (fused[..., :hq * d].unflatten(-1, (hq, d)),
            fused[..., hq * d:(hq + hkv) * d].unflatten(-1, (hkv, d)))


CASES = [
    # head_dim, rotary_dim, interleaved, batch, tokens, heads, key heads, scaling
    (64, 64, False, 2, 37, 16, 8, {}),
    (64, 64, True, 1, 1, 4, 4, {}),
    (64, 32, False, 3, 5, 12, 4, {"scaling": "linear", "factor": 4.0}),
    (64, 16, True, 1, 130, 8, 1, {"scaling": "base", "factor": 2.0}),
    (128, 128, False, 2, 65, 32, 8, {"scaling": "bands", "factor": 8.0, "original_length": 8192}),
    (128, 32, True, 1, 257, 3, 1, {"scaling": "ramp", "factor": 8.0, "original_length": 4096}),
    (96, 24, False, 2, 19, 5, 5, {}),     # 12 pairs: vectors of four
    (80, 10, True, 1, 33, 7, 1, {}),      # five pairs: one by one
    (6, 2, False, 2, 9, 3, 3, {}),
    (256, 256, True, 1, 17, 2, 2, {}),
    (1024, 64, False, 1, 3, 6, 2, {}),    # a token wider than a workgroup's round
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"d{c[0]}r{c[1]}{'i' if c[2] else 'h'}")
def test_rotate_and_its_gradient(case, dtype, device):
    d, r, inter, b, t, hq, hkv, scaling = case
    say("rotate", dtype, case)
    rot = rotary.Rotary(d, theta=1e6, rotary_dim=r, interleaved=inter, **scaling)
    q, k = (x.detach().requires_grad_() for x in _qk(dtype, (b, t), hq, hkv, d, device, d + t))
    rng = np.random.default_rng(t)
    pos = torch.tensor(rng.integers(0, 200000, size=(b, t)).astype(np.int32), device=device)
    qo, ko = rotary.rotate(q, k, rot, pos)
    for got, x in ((qo, q), (ko, k)):
        close(got, *turned(x.detach(), pos, rot), "forward")
        # the dims that do not rotate are copied
        assert torch.equal(got[..., r:], x[..., r:])
    g = torch.Generator(device=device).manual_seed(9)
    dq = torch.randn(qo.shape, generator=g, device=device).to(dtype)
    dk = torch.randn(ko.shape, generator=g, device=device).to(dtype)
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    close(gq, *turned(dq, pos, rot, back=True), "dq")
    close(gk, *turned(dk, pos, rot, back=True), "dk")


def test_gradient_against_differences(device):
    # the rotation is linear: <g, R(x + h) - R(x)> = <R^T g, h> up to the roundings of both
    rot = rotary.Rotary(64, rotary_dim=48, interleaved=True, scaling="ramp", factor=4.0,
                        original_length=4096)
    q, k = _qk(torch.float32, (2, 11), 4, 2, 64, device)
    h, g = torch.randn_like(q), torch.randn_like(q)
    x = q.detach().requires_grad_()
    y, _ = rotary.rotate(x, None, rot)
    (grad,) = torch.autograd.grad(y, x, g)
    with torch.no_grad():
        moved, _ = rotary.rotate(q + h, None, rot)
    left = (g.double() * (moved.double() - y.detach().double())).sum().item()
    right = (grad.double() * ((q + h).double() - q.double())).sum().item()
    # every element of y and of the gradient is within 10 half steps of float32 of the sums of
    # its pair (|.| <= 2 * 5.5 * magnitude here), all of the same sign at worst
    n = q.numel()
    size = 10 * 2.0 ** -24 * rot.magnitude
    worst = size * (2 * 22 * g.abs().max() + 22 * h.abs().max()).item() * n
    assert abs(left - right) <= worst
    assert worst < 0.05 * abs(g.double().norm() * h.double().norm()).item()


@pytest.mark.parametrize("positions", ["none", "scalar", "row", "batch", "far", "negative"])
def test_position_forms(positions, device):
    rot = rotary.Rotary(64, theta=1e4)
    q, k = _qk(torch.float32, (2, 21), 4, 2, 64, device)
    given, full = {
        "none": (None, torch.arange(21).expand(2, 21)),
        "scalar": (7, torch.full((2, 21), 7)),
        "row": (torch.arange(21) + 100, (torch.arange(21) + 100).expand(2, 21)),
        "batch": (torch.arange(42).view(2, 21), torch.arange(42).view(2, 21)),
        "far": (torch.arange(21) + (1 << 31) - 30, (torch.arange(21) + (1 << 31) - 30).expand(2, 21)),
        "negative": (torch.arange(21) - 1000, (torch.arange(21) - 1000).expand(2, 21)),
    }[positions]
    qo, ko = rotary.rotate(q, k, rot, given)
    if positions == "far":
        # float64 holds position * f to 2^31 * 2^-53 turns
        want, bound = turned(q, full, rot)
        close(qo, want, bound + 2.0 ** -20, positions)
    else:
        close(qo, *turned(q, full, rot), positions)
        close(ko, *turned(k, full, rot), positions)


def test_three_dimensions_and_no_key(device):
    rot = rotary.Rotary(64)
    q, k = _qk(torch.bfloat16, (45,), 6, 2, 64, device)
    pos = torch.arange(45, device=device, dtype=torch.int32) * 3
    qo, ko = rotary.rotate(q, k, rot, pos)
    close(qo, *turned(q, pos, rot), "q")
    alone, none = rotary.rotate(q, None, rot, pos)
    assert none is None and torch.equal(alone, qo)
    lone_k, _ = rotary.rotate(k, None, rot, pos)
    assert torch.equal(lone_k, ko)
    first, _ = rotary.rotate(q, None, rot)
    close(first, *turned(q, torch.arange(45), rot), "positions 0 .. N-1")


@pytest.mark.parametrize("how", ["transposed", "odd offset", "expanded", "sliced heads"])
def test_views_of_any_strides(how, device):
    rot = rotary.Rotary(64)
    g = torch.Generator(device=device).manual_seed(3)
    if how == "transposed":  # heads before tokens
        q = torch.randn(2, 4, 17, 64, generator=g, device=device).bfloat16().transpose(1, 2)
    elif how == "odd offset":  # rows that no 16-byte load fits
        q = torch.randn(2 * 17 * 4 * 64 + 1, generator=g, device=device).bfloat16()[1:].view(2, 17, 4, 64)
    elif how == "expanded":
        q = torch.randn(1, 17, 4, 64, generator=g, device=device).bfloat16().expand(2, 17, 4, 64)
    else:
        q = torch.randn(2, 17, 8, 64, generator=g, device=device).bfloat16()[:, :, ::2]
    qo, _ = rotary.rotate(q, None, rot)
    close(qo, *turned(q, torch.arange(17).expand(2, 17), rot), how)
    assert qo.is_contiguous()


def test_large_batch_takes_the_wide_form(device):
    rot = rotary.Rotary(64, theta=1e6)
    q, k = _qk(torch.bfloat16, (4, 4096), 16, 8, 64, device)
    qo, ko = rotary.rotate(q, k, rot)
    # the same rows a few at a time
    for at in (0, 1000, 4090):
        a, b = rotary.rotate(q[:, at:at + 6], k[:, at:at + 6], rot, torch.arange(at, at + 6))
        assert torch.equal(qo[:, at:at + 6], a) and torch.equal(ko[:, at:at + 6], b)


def test_one_gradient_of_two(device):
    rot = rotary.Rotary(64)
    q, k = (x.detach().requires_grad_() for x in _qk(torch.float32, (1, 9), 4, 2, 64, device))
    qo, ko = rotary.rotate(q, k, rot)
    (dq,) = torch.autograd.grad(qo, q, torch.ones_like(qo), retain_graph=True)
    close(dq, *turned(torch.ones(1, 9, 4, 64), torch.arange(9)[None], rot, back=True), "dq alone")
    (dk,) = torch.autograd.grad(ko, k, torch.ones_like(ko))
    close(dk, *turned(torch.ones(1, 9, 2, 64), torch.arange(9)[None], rot, back=True), "dk alone")


def test_replayed_graph_and_other_stream(device):
    rot = rotary.Rotary(64, scaling="linear", factor=2.0)
    q, k = _qk(torch.bfloat16, (2, 33), 4, 2, 64, device)
    q, k = q.contiguous(), k.contiguous()
    pos = torch.arange(66, device=device, dtype=torch.int32).view(2, 33)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rotary.rotate(q, k, rot, pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo, ko = rotary.rotate(q, k, rot, pos)
    for i in range(3):
        q.normal_()
        pos.add_(17)
        graph.replay()
        torch.cuda.synchronize()
        eq, ek = rotary.rotate(q, k, rot, pos)
        assert torch.equal(qo, eq) and torch.equal(ko, ek), i


def test_replayed_backward(device):
    """Forward and backward captured together, replayed, against eager passes."""
    rot = rotary.Rotary(64, rotary_dim=32, interleaved=True)
    q, k = _qk(torch.bfloat16, (2, 40), 4, 2, 64, device)
    q, k = (x.contiguous().requires_grad_() for x in (q, k))
    wq, wk = torch.randn_like(q), torch.randn_like(k)

    def grads():
        qo, ko = rotary.rotate(q, k, rot)
        return torch.autograd.grad((qo, ko), (q, k), (wq, wk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dq, dk = grads()
    for i in range(3):
        wq.normal_()
        wk.normal_()
        graph.replay()
        torch.cuda.synchronize()
        eq, ek = grads()
        assert torch.equal(dq, eq) and torch.equal(dk, ek), i


def test_only_what_needs_a_gradient_gets_one(device):
    rot = rotary.Rotary(64)
    q, k = _qk(torch.float32, (2, 5), 4, 2, 64, device)
    q, k = q.contiguous().requires_grad_(), k.contiguous()
    qo, ko = rotary.rotate(q, k, rot)
    (qo.sum() + ko.sum()).backward()
    assert k.grad is None
    close(q.grad, *turned(torch.ones(2, 5, 4, 64), torch.arange(5).expand(2, 5), rot, back=True), "dq")
    # an expanded key: one head's gradient is the sum over its copies
    one = torch.randn(2, 5, 1, 64, device=device, requires_grad=True)
    _, ko = rotary.rotate(q.detach(), one.expand(2, 5, 3, 64), rot)
    ko.sum().backward()
    want, bound = turned(torch.ones(2, 5, 1, 64), torch.arange(5).expand(2, 5), rot, back=True)
    close(one.grad, 3 * want, 3 * bound + 2 * 2.0 ** -24 * 3 * abs(want), "shared")


def test_gradient_of_a_gradient(device):
    """The backward is linear in the incoming gradient: its own backward turns forward again."""
    rot = rotary.Rotary(64, rotary_dim=48)
    q, k = _qk(torch.float32, (1, 7), 3, 3, 64, device)
    q, k = (x.contiguous().requires_grad_() for x in (q, k))
    g = torch.Generator(device=device).manual_seed(5)
    wq, wk, uq, uk = (torch.randn(q.shape, generator=g, device=device) for _ in range(4))
    wq.requires_grad_()
    qo, ko = rotary.rotate(q, k, rot)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (wq, wk), create_graph=True)
    (ddq,) = torch.autograd.grad((dq * uq).sum() + (dk * uk).sum(), (wq,))
    close(ddq, *turned(uq, torch.arange(7)[None], rot), "second")
    # and the gradients are not functions of what was rotated
    dq, _ = torch.autograd.grad(rotary.rotate(q, k, rot), (q, k), (wq, wk), create_graph=True)
    assert torch.autograd.grad(dq.sum(), (q,), allow_unused=True) == (None,)
