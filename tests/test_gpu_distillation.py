"""The distillation loss and its gradient against their definition in float64."""

import math

import pytest
import torch

import _ends
from _helpers import say
from mfattn.kernels import distillation

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]


def _operands(dtype, rows, v, k, device, *, seed=0, temperature=1.0, total=False, spread=2.0):
    g = torch.Generator(device=device).manual_seed(seed + 31 * rows + 7 * v + k)
    z = (spread * torch.randn(rows, v, generator=g, device=device))
    ids = torch.rand(rows, v, generator=g, device=device).argsort(1)[:, :k].contiguous()
    t = 5 + 2 * torch.randn(rows, k, generator=g, device=device)
    z.scatter_add_(1, ids, 0.8 * t)
    z, t = z.to(dtype), t.to(dtype)
    more = {"temperature": temperature}
    if total:
        more["teacher_total"] = torch.logsumexp(t.float() / temperature, 1) + 0.3 * torch.rand(
            rows, generator=g, device=device) + 0.01
    return z, t, ids, more


def _check(z, t, ids, more, upstream=None):
    """The three ways to the loss and both to the gradient."""
    v = z.shape[-1]
    rows = z.numel() // v
    flat = (z.reshape(rows, v), t.reshape(rows, -1), ids.reshape(rows, -1), more["temperature"],
            *(None if more.get(n) is None else more[n].reshape(-1) for n in ("teacher_total", "weights")))
    with torch.no_grad():
        alone = distillation.top_logits_loss(z, t, ids, **more)
        loss, grad = distillation.top_logits_loss_and_gradient(z, t, ids, **more)
    want = _ends.distill(*flat)
    assert alone.shape == z.shape[:-1] and alone.dtype is torch.float32
    _ends.check(alone.reshape(-1), *want[:2], "loss")
    _ends.check(loss.reshape(-1), *want[:2], "loss beside the gradient")
    _ends.check(grad.reshape(rows, v), *want[2:], "gradient in one pass")
    leaf = z.detach().requires_grad_()
    recorded = distillation.top_logits_loss(leaf, t, ids, **more)
    assert torch.equal(recorded, alone)
    if upstream is None:
        upstream = torch.linspace(-1, 2, rows, device=z.device).view(alone.shape)
    (g,) = torch.autograd.grad(recorded, leaf, upstream)
    want = _ends.distill(*flat, upstream.reshape(-1))
    _ends.check(g.reshape(rows, v), *want[2:], "gradient by the backward pass")
    return loss, grad, g


# less than a vector, one workgroup's, two and more vectors a thread, beyond the registers, the most
VOCABULARIES = [1, 5, 8, 100, 1023, 8192, 8193, 20000, 65536, 65541, 131072, 131080, 140001, 393216]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", VOCABULARIES)
@pytest.mark.parametrize("total", [False, True], ids=["softmax", "total"])
def test_vocabularies(v, dtype, total, device):
    say("distill", v, dtype, total)
    _check(*_operands(dtype, 3, v, min(v, 37), device, temperature=1.5, total=total))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [1, 2, 63, 64, 65, 200, 1024])
@pytest.mark.parametrize("total", [False, True], ids=["softmax", "total"])
def test_entries(k, dtype, total, device):
    say("distill entries", k, dtype, total)
    _check(*_operands(dtype, 5, 1500, k, device, temperature=0.7, total=total))


# rows of 256 threads: two, one and half of their ranges, and the first row too long for them
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [3, 4096, 8193, 16389, 32771, 32776])
@pytest.mark.parametrize("total", [False, True], ids=["softmax", "total"])
def test_more_rows_than_are_taken_at_once(v, dtype, total, device):
    say("distill rows", v, dtype, total)
    z, t, ids, more = _operands(dtype, 515, v, min(v, 70), device, temperature=1.5, total=total)
    _check(z, t, ids, more)


@pytest.mark.parametrize("rows", [1, 2, 300, 5000])
def test_rows(rows, device):
    z, t, ids, more = _operands(torch.bfloat16, rows, 333, 8, device, total=True)
    _check(z, t, ids, more)


def test_shapes_types_and_weights(device):
    z, t, ids, more = _operands(torch.bfloat16, 24, 999, 12, device, temperature=2.0, total=True)
    weights = torch.rand(24, device=device)
    weights[::3] = 0
    more = {"temperature": 2.0, "teacher_total": more["teacher_total"].view(2, 3, 4),
            "weights": weights.view(2, 3, 4)}
    shape = (2, 3, 4)
    base = _check(z.view(*shape, -1), t.view(*shape, -1), ids.view(*shape, -1), more)
    for kind in (torch.int32, torch.int16):
        same = _check(z.view(*shape, -1), t.view(*shape, -1), ids.view(*shape, -1).to(kind), more)
        assert all(torch.equal(a, b) for a, b in zip(base, same))
    # a float32 teacher of a bfloat16 student, and double weights
    more["weights"] = more["weights"].double()
    same = _check(z.view(*shape, -1), t.view(*shape, -1).float(), ids.view(*shape, -1), more)
    assert all(torch.equal(a, b) for a, b in zip(base, same))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_weight_hold_anything(dtype, device):
    z, t, ids, more = _operands(dtype, 12, 2000, 16, device, total=True)
    more["weights"] = torch.ones(12, device=device)
    more["weights"][::2] = 0
    clean = _check(z, t, ids, more)
    z[::2] = float("nan")
    t[0] = float("inf")
    ids[2] = 77
    more["teacher_total"][4] = float("nan")
    got = _check(z, t, ids, more)
    assert all(torch.equal(a, b) for a, b in zip(clean, got))
    for x in got:
        assert not x[::2].any()
    # nor where nothing comes from above
    up = torch.zeros(12, device=device)
    assert not _check(z, t, ids, more, up)[2].any()


@pytest.mark.parametrize("total", [False, True], ids=["softmax", "total"])
def test_entries_that_are_not_there(total, device):
    z, t, ids, more = _operands(torch.float32, 9, 700, 10, device, total=total)
    ids[1, 5:] = -1
    ids[2, :9] = -7
    ids[3, ::2] = 700
    ids[4, 1] = 1 << 40
    ids[5] = -1                # none at all
    t[6, 3] = -math.inf        # there, without mass
    t[7] = -math.inf
    t[8, 1:] = torch.finfo(torch.float32).min
    loss, grad, g = _check(z, t, ids, more)
    if not total:
        assert loss[5] == 0 and not grad[5].any() and not g[5].any()
        assert loss[7] == 0 and not grad[7].any()
        z[5] = float("nan")
        loss, grad, g = _check(z, t, ids, more)
        assert not grad[5].any() and not g[5].any()


@pytest.mark.parametrize("total", [False, True], ids=["softmax", "total"])
def test_the_same_id_more_than_once(total, device):
    z, t, ids, more = _operands(torch.float32, 6, 400, 20, device, total=total)
    ids[:, 7] = ids[:, 3]
    ids[:, 19] = ids[:, 3]
    ids[4] = 11
    _check(z, t, ids, more)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("total", [False, True], ids=["softmax", "total"])
def test_logits_that_are_masked(dtype, total, device):
    z, t, ids, more = _operands(dtype, 8, 1200, 6, device, total=total)
    low = torch.finfo(dtype).min
    free = torch.ones(8, 1200, dtype=torch.bool, device=device).scatter_(1, ids, False)
    half = free & (torch.arange(1200, device=device) % 2 == 0)
    z[0][half[0]] = -math.inf
    z[1][half[1]] = low
    z[2][: 600] = torch.where(free[2][:600], -math.inf, z[2][:600])
    z[3] = low                     # all the same: uniform
    if not total:
        z[4][free[4]] = -math.inf  # the entries alone
        z[5][free[5]] = low
    _check(z, t, ids, more)
    # an entry that the student rules out costs everything, and its gradient is finite
    z[6, ids[6, 2]] = -math.inf
    loss, grad = distillation.top_logits_loss_and_gradient(z, t, ids, **more)
    assert loss[6] == math.inf and grad.isfinite().all()
    # what is not a number, and a row of nothing, stay in their row
    nothing = torch.full((1200,), -math.inf, device=device, dtype=dtype)
    for where, value in ((33, float("nan")), (33, math.inf), (slice(None), nothing)):
        bad = z.clone()
        bad[7, where] = value
        got, dgot = distillation.top_logits_loss_and_gradient(bad, t, ids, **more)
        assert got[7].isnan() and dgot[7].isnan().any()
        assert torch.equal(got[:7], loss[:7]) and torch.equal(dgot[:7], grad[:7])
    for value in (float("nan"), math.inf):
        odd = t.clone()
        odd[7, 2] = value
        got, dgot = distillation.top_logits_loss_and_gradient(z, odd, ids, **more)
        assert got[7].isnan() and dgot[7].isnan().all()
        assert torch.equal(got[:7], loss[:7]) and torch.equal(dgot[:7], grad[:7])


def test_a_confident_student_beyond_the_entries(device):
    # what is left beyond the entries is e^-30 of the student's mass: far below the rounding of
    # a sum of all, and the loss lives on its logarithm
    z, t, ids, more = _operands(torch.float32, 4, 3000, 5, device, total=True, spread=0.5)
    z.scatter_add_(1, ids, torch.full_like(t, 30.0))
    _check(z, t, ids, more)


def test_a_total_below_the_entries(device):
    # entries that have more than the whole: nothing is left, their masses count as they are
    z, t, ids, more = _operands(torch.float32, 4, 500, 5, device, total=True)
    more["teacher_total"] = more["teacher_total"] - 0.5
    _check(z, t, ids, more)


def test_every_id_an_entry(device):
    z, t, ids, more = _operands(torch.float32, 3, 64, 64, device)
    _check(z, t, ids, more)
    more["teacher_total"] = torch.logsumexp(t, 1) - 0.01  # (nothing left)
    _check(z, t, ids, more)


@pytest.mark.parametrize("how", ["padded vocabulary", "odd offset", "transposed", "batch"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_views_of_any_strides(how, dtype, device):
    z, t, ids, more = _operands(dtype, 12, 600, 7, device, total=True)
    wide = torch.full((12, 800), float("nan"), device=device, dtype=dtype)
    if how == "padded vocabulary":
        wide[:, :600] = z
        z = wide[:, :600]
    elif how == "odd offset":
        wide[:, 101:701] = z
        z = wide[:, 101:701]
    elif how == "transposed":
        z = z.t().contiguous().t()
    else:
        z, t, ids = (x.view(3, 4, -1).transpose(0, 1) for x in (z, t, ids))
        more["teacher_total"] = more["teacher_total"].view(3, 4).t()
    _check(z, t, ids, more)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [100, 5001, 65536, 100000, 140001])
def test_in_the_logits_place(v, dtype, device):
    z, t, ids, more = _operands(dtype, 5, v, 9, device, total=True)
    loss, grad = distillation.top_logits_loss_and_gradient(z, t, ids, **more)
    other = torch.empty_like(z)
    loss2, same = distillation.top_logits_loss_and_gradient(z, t, ids, out=other, **more)
    assert same is other and torch.equal(other, grad) and torch.equal(loss, loss2)
    # rows of a padded projection, what is beside them left as it is
    wide = torch.full((5, v + 50), 7.0, device=device, dtype=dtype)
    wide[:, 10:10 + v] = z
    version = wide._version
    loss3, same = distillation.top_logits_loss_and_gradient(wide[:, 10:10 + v], t, ids,
                                                            out=wide[:, 10:10 + v], **more)
    assert torch.equal(same, grad) and torch.equal(loss, loss3)
    assert (wide[:, :10] == 7).all() and (wide[:, 10 + v:] == 7).all()
    assert wide._version > version


def test_outputs_that_are_refused(device):
    z, t, ids, more = _operands(torch.float32, 5, 90, 9, device)
    call = distillation.top_logits_loss_and_gradient
    wide = torch.zeros(5, 100, device=device)
    for out, match in ((torch.empty(5, 91, device=device), "out must be"),
                       (torch.empty(5, 90, device=device).bfloat16(), "out must be"),
                       (torch.empty(90, 5, device=device).t(), "evenly spaced"),
                       (torch.empty(5, 90, device=device, requires_grad=True), "require a gradient"),
                       (torch.empty(5, 90), "out must be")):
        with pytest.raises(ValueError, match=match):
            call(z, t, ids, out=out, **more)
    with pytest.raises(ValueError, match="share no memory"):
        call(wide[:, :90], t, ids, out=wide[:, 5:95], **more)
    # the teacher or the weights beside the gradient
    wide[:, 90:99] = t
    with pytest.raises(ValueError, match="teacher or the weights"):
        call(z, wide.view(-1)[455:500].view(5, 9), ids, out=wide.view(-1)[:450].view(5, 90), **more)
    with pytest.raises(ValueError, match="teacher or the weights"):
        call(z, t, ids, weights=wide.view(-1)[495:], out=wide.view(-1)[:450].view(5, 90))
    empty = torch.empty(0, 90, device=device)
    assert call(empty, t[:0], ids[:0], out=empty)[1] is empty


def test_zero_rows(device):
    z = torch.zeros(0, 50, device=device, requires_grad=True)
    t, ids = torch.zeros(0, 4, device=device), torch.zeros(0, 4, dtype=torch.int64, device=device)
    loss = distillation.top_logits_loss(z, t, ids)
    assert loss.shape == (0,)
    (g,) = torch.autograd.grad(loss.sum(), z)
    assert g.shape == z.shape
    loss, g = distillation.top_logits_loss_and_gradient(z.detach(), t, ids)
    assert loss.shape == (0,) and g.shape == z.shape


def test_offsets_past_two_gigabytes(device):
    # more than 2^31 logits: the last rows against the same rows alone
    rows, v = 17000, 131072
    z = torch.empty(rows, v, device=device, dtype=torch.bfloat16)
    z[-3:] = torch.randn(3, v, device=device).bfloat16()
    t = torch.randn(rows, 4, device=device)
    ids = torch.randint(0, v, (rows, 4), device=device)
    weights = torch.zeros(rows, device=device)
    weights[-3:] = 1
    loss, grad = distillation.top_logits_loss_and_gradient(z, t, ids, weights=weights, out=z.clone())
    some, dsome = distillation.top_logits_loss_and_gradient(z[-3:].clone(), t[-3:], ids[-3:])
    assert torch.equal(loss[-3:], some) and torch.equal(grad[-3:], dsome)
    assert not loss[:-3].any() and not grad[:-3].any()


def test_gradient_against_differences(device):
    # phi(h) = sum of losses at z + h dz, float64 differences of the definition against the
    # kernel's gradient, and the kernel's own differences against both
    z, t, ids, more = _operands(torch.float32, 6, 300, 8, device, temperature=1.3, total=True)
    dz = torch.randn_like(z)
    _, grad = distillation.top_logits_loss_and_gradient(z, t, ids, **more)
    slope = (grad.double() * dz.double()).sum().item()

    def exact(h):
        return _ends.distill(z.double() + h * dz.double(), t, ids, 1.3,
                             more["teacher_total"])[0].sum().item()

    def phi(h):
        return distillation.top_logits_loss((z + h * dz), t, ids, **more).double().sum().item()

    tiny, h = 2.0 ** -14, 2.0 ** -4
    fine = (exact(tiny) - exact(-tiny)) / (2 * tiny)
    assert abs(fine - slope) <= 1e-5 * (grad.abs().double() * dz.abs().double()).sum().item()
    # float32 inputs move the logits by E |z|, whose slopes are bounded by the gradient's size
    bound = _ends.distill(z, t, ids, 1.3, more["teacher_total"])[1].sum().item()
    noise = (bound + 4 * _ends.E * (grad.abs().double() * (z.abs() + dz.abs()).double()).sum().item()) / h
    formula = abs((exact(h) - exact(-h)) / (2 * h) - fine)
    assert abs((phi(h) - phi(-h)) / (2 * h) - slope) <= formula * 1.01 + 2 * noise


def test_graphs_of_the_backward_pass_are_refused(device):
    z, t, ids, more = _operands(torch.float32, 2, 30, 3, device)
    loss = distillation.top_logits_loss(z.requires_grad_(), t, ids, **more)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(loss.sum(), z, create_graph=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [700, 9000, 65536, 140001])
@pytest.mark.parametrize("total", [False, True], ids=["softmax", "total"])
def test_largest_logits_far_behind_the_first(v, dtype, total, device):
    """Exponentials are taken beside a logit near the front: what lies hundreds of units above or
    below it further on, in one place, in many or nowhere, counts as the definition says."""
    z, t, ids, more = _operands(dtype, 10, v, 5, device, total=total)
    low = torch.finfo(dtype).min
    half = v // 2
    z[0, half:] += 300            # exp overflows beside the first
    z[1, :half] += 300            # and vanishes
    z[2, -1] = 500
    z[3, ::997] += 200
    z[4, :half] = -math.inf
    z[5, :half] = low
    z[6] -= 1000
    z[7] = torch.linspace(-400, 400, v, device=device).to(dtype)
    z[8] = torch.linspace(400, -400, v, device=device).to(dtype)
    z[9, :-1] = -math.inf
    for r in range(10):           # entries that the student does not rule out
        z[r, ids[r]] = z[r][z[r].float().argmax()].clone()
    _check(z, t, ids, more)
    more["temperature"] = 0.1
    if total:
        more["teacher_total"] = torch.logsumexp(t.float() / 0.1, 1) + 0.2
    _check(z, t, ids, more)
