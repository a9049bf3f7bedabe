"""The distillation loss where the student has next to nothing beyond the teacher's entries: its
mass there is far below what float32 holds beside the row's largest logit."""

import math

import pytest
import torch

import _ends
from _helpers import say
from _ends import E
from mfattn.kernels import distillation

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]


def _definition(z, teacher, ids, temperature, total, upstream=None):
    """(loss, bound, gradient, bound) row by row, the remainder's mass by its logarithm."""
    rows, v = z.shape
    z, t = z.double().cpu() / temperature, teacher.double().cpu() / temperature
    ids, total = ids.cpu().long(), total.double().cpu()
    loss, loss_e = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    grad, grad_e = torch.zeros_like(z), torch.zeros_like(z)
    for n in range(rows):
        here = (ids[n] >= 0) & (ids[n] < v)
        at, logp = ids[n][here], t[n][here] - total[n]
        p = logp.exp()
        rest = max(0.0, 1 - float(p.sum()))
        mass = float(p.sum()) + rest
        beyond = torch.ones(v, dtype=torch.bool)
        beyond[at] = False
        logq = torch.log_softmax(z[n], 0)
        q = logq.exp()
        logs = float(torch.logsumexp(logq[beyond], 0)) if beyond.any() else -math.inf
        # the student's masses beyond the entries, beside their own sum
        share = torch.zeros(v, dtype=torch.float64)
        if logs > -math.inf:
            share[beyond] = torch.softmax(z[n][beyond], 0)
        kl = float(torch.where(p > 0, p * (logp - logq[at]), 0.0).sum())
        if rest > 0:
            kl += rest * (math.log(rest) - logs)
        loss[n] = temperature ** 2 * kl
        # an exponential's argument has three roundings and the exponential two steps; a thread
        # (one of 256 at least) adds its part of the row, then 6 + 16 sums
        arg = torch.where(z[n] > -math.inf, z[n].max() - z[n], 0.0)
        own = torch.where(beyond, z[n], -math.inf)
        arg_own = torch.where(own > -math.inf, own.max() - own, 0.0) if logs > -math.inf else 0 * arg
        depth = v // 256 + 8 + 22 + 4
        sums = (depth + 3 * float((q * arg).sum())) * E
        rest_sums = (depth + 3 * float((share * arg_own).sum())) * E
        loss_e[n] = temperature ** 2 * (mass * sums + rest * (sums + rest_sums)) + 2 * E * abs(float(loss[n]))
        w = temperature * (1.0 if upstream is None else float(upstream[n]))
        named = torch.zeros(v, dtype=torch.float64).index_add_(0, at, p)
        grad[n] = w * (q * mass - named - rest * share)
        # exponentials below 2^-126 are zero: beside a sum of at least one, both times
        grad_e[n] = abs(w) * (q * mass * ((3 * arg + 8) * E + sums)
                              + named * 6 * E * max(1, len(at) ** 0.5)
                              + rest * share * ((3 * arg_own + 8) * E + rest_sums)
                              + 2.0 ** -125 * (mass + rest))
    return loss, loss_e, grad, grad_e


def _check(z, t, ids, total, temperature):
    more = {"temperature": temperature, "teacher_total": total}
    want = _definition(z, t, ids, temperature, total)
    loss, grad = distillation.top_logits_loss_and_gradient(z, t, ids, **more)
    _ends.check(loss, *want[:2], "loss beside the gradient")
    _ends.check(grad, *want[2:], "gradient in one pass")
    place = z.clone()
    again, same = distillation.top_logits_loss_and_gradient(place, t, ids, out=place, **more)
    assert torch.equal(again, loss) and torch.equal(same, grad)
    leaf = z.detach().requires_grad_()
    alone = distillation.top_logits_loss(leaf, t, ids, **more)
    _ends.check(alone.detach(), *want[:2], "loss")
    up = torch.linspace(-1, 2, len(z), device=z.device)
    (g,) = torch.autograd.grad(alone, leaf, up)
    want = _definition(z, t, ids, temperature, total, up)
    _ends.check(g, *want[2:], "gradient by the backward pass")
    return loss, grad


def _operands(dtype, rows, v, k, gap, temperature, device):
    """Entries that lie ``gap * temperature`` above every other logit, and a teacher that has a
    tenth beyond its entries (in the first row next to nothing)."""
    g = torch.Generator(device=device).manual_seed(rows + 7 * v + k + int(gap))
    z = temperature * torch.randn(rows, v, generator=g, device=device).clamp(-4, 4)
    ids = torch.rand(rows, v, generator=g, device=device).argsort(1)[:, :k].contiguous()
    t = temperature * torch.randn(rows, k, generator=g, device=device)
    z.scatter_(1, ids, temperature * (gap + 8 + torch.rand(rows, k, generator=g, device=device)))
    z, t = z.to(dtype), t.to(dtype)
    total = torch.logsumexp(t.float() / temperature, 1) + 0.1
    total[0] -= 0.1
    return z, t, ids, total


# where 64 and more such exponentials begin to vanish, where all have, and where 64 bits lose them
@pytest.mark.parametrize("gap", [60, 76, 80, 84, 89, 120, 200, 900, 20000])
@pytest.mark.parametrize("temperature", [1.0, 0.1, 4.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_entries_far_above_the_rest(dtype, temperature, gap, device):
    say("distill tails", dtype, temperature, gap)
    z, t, ids, total = _operands(dtype, 4, 1000, 5, gap, temperature, device)
    loss, _ = _check(z, t, ids, total, temperature)
    assert loss.isfinite().all()
    # a tenth of the teacher's mass costs what its logarithm says, whatever the gap
    assert (loss[1:] > 0.09 * temperature ** 2 * gap).all()


# rows of 256, 512 and 1024 threads, in registers and read again; odd values behind the vectors
@pytest.mark.parametrize("rows, v", [(3, 7), (3, 8193), (3, 65541), (3, 131077), (3, 140001),
                                     (515, 4099), (515, 16389)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_entries_far_above_the_rest_in_every_variant(rows, v, dtype, device):
    say("distill tails", rows, v, dtype)
    _check(*_operands(dtype, rows, v, min(v - 2, 70), 150, 1.0, device), 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_largest_of_the_rest_anywhere(dtype, device):
    """One logit of the rest above the others: the first, the last of the row's whole vectors, behind
    them, beside an entry; and a rest that spans more than an exponential does."""
    v = 4099
    z, t, ids, total = _operands(dtype, 7, v, 6, 300, 1.0, device)
    ids[:] = torch.tensor([3, 9, 1000, 2000, 4093, 4097], device=device)
    z = torch.randn(7, v, device=device)
    for row, at in enumerate((0, 4095, 4098, 8, 4096)):
        z[row, at] = 120
    z[5] = torch.linspace(-300, 0, v, device=device)
    z[6] = torch.linspace(0, -300, v, device=device)
    z.scatter_(1, ids, 400 + torch.rand(7, 6, device=device))
    _check(z.to(dtype), t, ids, total, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_entries_named_twice(dtype, device):
    z, t, ids, total = _operands(dtype, 5, 2000, 200, 100, 1.0, device)
    ids[1, 70:] = ids[1, :130].clone()
    ids[2] = ids[2, 0]
    ids[3, 64] = ids[3, 3]
    ids[4, ::2] = -1
    z[1:3] = z[1:3].clamp(max=30.0)  # (the former entries above the rest no more)
    loss, grad = _check(z, t, ids, total, 1.0)
    for _ in range(3):
        again = distillation.top_logits_loss_and_gradient(z, t, ids, teacher_total=total)
        assert torch.equal(again[0], loss) and torch.equal(again[1], grad)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_rest_of_minus_infinity(dtype, device):
    """Without mass beyond the entries a teacher that has some there costs everything; a teacher
    that has none costs what its entries do."""
    z, t, ids, total = _operands(dtype, 4, 1003, 6, 0, 1.0, device)
    none = torch.full_like(z, -math.inf).scatter_(1, ids, z.gather(1, ids))
    none[2:] -= 2000
    total[1::2] = torch.logsumexp(t.float(), 1)[1::2] - 0.01
    loss, grad = _check(none, t, ids, total, 1.0)
    assert loss[2] == math.inf and loss[1::2].isfinite().all() and grad.isfinite().all()
    # entries that the student rules out, beside a rest that it does not
    low = z.clone().scatter_(1, ids, torch.full_like(t, -math.inf))
    loss, grad = _check(low, t, ids, total, 1.0)
    assert (loss == math.inf).all() and grad.isfinite().all()


def test_what_is_not_a_number_among_entries_and_rest(device):
    z, t, ids, total = _operands(torch.float32, 6, 1003, 6, 100, 1.0, device)
    clean = distillation.top_logits_loss_and_gradient(z, t, ids, teacher_total=total)
    at = int(ids[3, 2])
    free = next(i for i in range(1003) if i not in ids[3].tolist())
    for where in (at, free):
        for value in (math.nan, math.inf):
            bad = z.clone()
            bad[3, where] = value
            loss, grad = distillation.top_logits_loss_and_gradient(bad, t, ids, teacher_total=total)
            assert loss[3].isnan() and grad[3].isnan().any()
            keep = [0, 1, 2, 4, 5]
            assert torch.equal(loss[keep], clean[0][keep]) and torch.equal(grad[keep], clean[1][keep])


def test_gradient_against_differences_of_the_definition(device):
    z, t, ids, total = _operands(torch.float32, 3, 200, 4, 95, 1.0, device)
    dz = torch.randn_like(z)
    _, grad = distillation.top_logits_loss_and_gradient(z, t, ids, teacher_total=total)
    h = 2.0 ** -14

    def phi(s):
        return _definition(z.double() + s * dz.double(), t, ids, 1.0, total)[0].sum().item()

    slope = (grad.double() * dz.double()).sum().item()
    # the difference is off by h^2 / 6 of a third derivative of some units and by 2^-52 of the
    # losses (some tens) over h; the gradient by its float32 terms
    room = 1e-6 * (grad.abs() * dz.abs()).sum().item() + 1e-8
    assert abs((phi(h) - phi(-h)) / (2 * h) - slope) <= room
