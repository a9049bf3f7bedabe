"""Layer norm and RMS norm against their definition in float64: widths, strides, gradients."""

import pytest
import torch

import _ends
from _helpers import say
from mfattn.kernels import normalization

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]
# one element, a lane group's end, a wave's, several vectors, a workgroup's, the most
WIDTHS = [1, 7, 8, 64, 127, 128, 129, 256, 511, 512, 771, 1024, 1025, 2048, 2056, 4096, 5000, 8192,
          16384]


def _operands(dtype, rows, dim, device, *, params=None, seed=0):
    g = torch.Generator(device=device).manual_seed(1000 * dim + rows + seed)
    x = torch.randn(rows, dim, generator=g, device=device) * (
        0.2 + 2 * torch.rand(rows, 1, generator=g, device=device)) + torch.randn(
        rows, 1, generator=g, device=device)
    params = params or dtype
    w = 1 + 0.3 * torch.randn(dim, generator=g, device=device)
    b = 0.3 * torch.randn(dim, generator=g, device=device)
    dy = torch.randn(rows, dim, generator=g, device=device)
    return x.to(dtype), w.to(params), b.to(params), dy.to(dtype)


def _check(x, w, b, dy, center, eps=1e-5):
    leaves = [t.detach().requires_grad_() for t in ((x, w, b) if center else (x, w))]
    y = normalization.layer_norm(*leaves, eps=eps) if center else \
        normalization.rms_norm(*leaves, eps=eps)
    grads = torch.autograd.grad(y, leaves, dy)
    d = x.shape[-1]
    want = _ends.norm(x.reshape(-1, d), w, b if center else None, eps, center, dy.reshape(-1, d))
    _ends.check(y.detach().reshape(-1, d), *want["y"], "y")
    _ends.check(grads[0].reshape(-1, d), *want["dx"], "dx")
    for name, g, p in zip(("dweight", "dbias"), grads[1:], leaves[1:]):
        assert g.dtype is p.dtype
        _ends.check(g, *want[name], name)
    with torch.no_grad():  # the same without a graph
        again = normalization.layer_norm(*leaves, eps=eps) if center else \
            normalization.rms_norm(*leaves, eps=eps)
    assert torch.equal(again, y)
    return y, grads


@pytest.mark.parametrize("center", [True, False], ids=["layer", "rms"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", WIDTHS)
@pytest.mark.parametrize("rows", [37, 1100], ids=["few", "many"])
def test_widths(rows, dim, dtype, center, device):
    say("norm", rows, dim, dtype, center)
    x, w, b, dy = _operands(dtype, rows, dim, device)
    _check(x, w, b, dy, center)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 63, 64, 65, 1023, 1024, 1025, 4097])
@pytest.mark.parametrize("dim", [64, 1024, 4096])
def test_rows(rows, dim, dtype, device):
    say("norm rows", rows, dim, dtype)
    _check(*_operands(dtype, rows, dim, device), True)


def test_float32_weights_of_bfloat16_rows(device):
    for dim in (256, 771, 4096):
        _check(*_operands(torch.bfloat16, 19, dim, device, params=torch.float32), True)
        _check(*_operands(torch.bfloat16, 19, dim, device, params=torch.float32), False)


@pytest.mark.parametrize("how", ["slice", "odd offset", "transposed", "expanded", "batch", "reversed dims"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_views_of_any_strides(how, dtype, device):
    x, w, b, dy = _operands(dtype, 12, 96, device)
    wide = torch.randn(12, 200, device=device).to(dtype)
    if how == "slice":
        x, dy = wide[:, 8:104], wide[:, 104:200]
    elif how == "odd offset":
        x, dy = wide[:, 3:99], wide[:, 101:197]
    elif how == "transposed":
        x = torch.randn(96, 12, device=device).to(dtype).t()
    elif how == "expanded":
        dy = dy[:1].expand(12, 96)
    elif how == "batch":
        x, dy = x.view(3, 4, 96).transpose(0, 1), dy.view(4, 3, 96)
    else:
        x = torch.randn(12, 2, 96, device=device).to(dtype)[:, 1]
    _check(x, w, b, dy, True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_whose_mean_is_large_beside_their_spread(dtype, device):
    x, w, b, dy = _operands(dtype, 9, 1024, device)
    x = (1000 + x.float()).to(dtype)
    _check(x, w, b, dy, True)
    # rows of one value: no spread but eps, and its root
    x = torch.full((3, 512), 3.5, device=device, dtype=dtype)
    y, grads = _check(x, w[:512], b[:512], dy[:3, :512], True)
    assert torch.equal(y, b[:512].expand(3, 512))


def test_zero_rows(device):
    x = torch.zeros(0, 4, 64, device=device, requires_grad=True)
    w, b = torch.ones(64, device=device, requires_grad=True), torch.ones(64, device=device, requires_grad=True)
    y = normalization.layer_norm(x, w, b)
    assert y.shape == x.shape
    for g, t in zip(torch.autograd.grad(y.sum(), (x, w, b)), (x, w, b)):
        assert g.shape == t.shape and not g.any()
    with torch.no_grad():
        assert normalization.rms_norm(x, w).shape == x.shape


def test_a_row_that_is_not_finite_stays_alone(device):
    x, w, b, dy = _operands(torch.float32, 40, 1024, device)
    clean, _ = _check(x, w, b, dy, True)
    for value in (float("nan"), float("inf"), -float("inf")):
        y = x.clone()
        y[7, 100] = value
        got = normalization.layer_norm(y, w, b)
        keep = torch.arange(40, device=device) != 7
        assert torch.equal(got[keep], clean[keep])
        assert got[7].isnan().any()


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 2), (1, 2)])
@pytest.mark.parametrize("rows", [300, 1300])
def test_gradients_that_are_asked_for(rows, which, device):
    x, w, b, dy = _operands(torch.bfloat16, rows, 1024, device)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = normalization.layer_norm(*leaves)
    every = torch.autograd.grad(y, leaves, dy)
    leaves = [t.detach().requires_grad_(i in which) for i, t in enumerate(leaves)]
    y = normalization.layer_norm(*leaves)
    some = torch.autograd.grad(y, [leaves[i] for i in which], dy)
    for i, g in zip(which, some):
        assert torch.equal(g, every[i])


def test_gradients_against_differences(device):
    # phi(h) = <dy, y(x + h dx, w + h dw, b + h db)>; its slope at 0 against (phi(h) - phi(-h)) / 2h,
    # off by h^2 times a third derivative and the roundings of y over h
    x, w, b, dy = _operands(torch.float32, 8, 256, device)
    tx, tw, tb = (torch.randn_like(t) for t in (x, w, b))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = normalization.layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    slope = sum((g.double() * t.double()).sum().item() for g, t in zip(grads, (tx, tw, tb)))

    def phi(h):
        moved = [(p + h * t).detach() for p, t in zip((x, w, b), (tx, tw, tb))]
        return (dy.double() * normalization.layer_norm(*moved).double()).sum().item()

    def exact(h):
        moved = [p.double() + h * t.double() for p, t in zip((x, w, b), (tx, tw, tb))]
        off = moved[0] - moved[0].mean(-1, keepdim=True)
        return (dy.double() * (off * ((off * off).mean(-1, keepdim=True) + 1e-5) ** -0.5 * moved[1]
                               + moved[2])).sum().item()

    h = 2.0 ** -6
    # what the formula itself leaves between the two, measured in 64 bits
    formula = abs((exact(h) - exact(-h)) / (2 * h) - (exact(2.0 ** -16) - exact(-2.0 ** -16)) / 2.0 ** -15)
    bound = _ends.norm(x, w, b, 1e-5, True)["y"][1] + 8 * _ends.E * (x.abs().double() + y.abs().double())
    noise = 4 * (dy.abs().double() * bound).sum().item() / (2 * h) * 2
    assert abs((phi(h) - phi(-h)) / (2 * h) - slope) <= formula + noise + 1e-3 * abs(slope)


def test_the_same_bits_every_time_and_on_another_stream(device):
    x, w, b, dy = _operands(torch.bfloat16, 5000, 1024, device)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    first = torch.autograd.grad(normalization.layer_norm(*leaves), leaves, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = torch.autograd.grad(normalization.layer_norm(*leaves), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(first, second):
        assert torch.equal(a, c)


def test_graphs_of_the_backward_pass_are_refused(device):
    x, w, b, dy = _operands(torch.float32, 4, 64, device)
    x.requires_grad_()
    for y in (normalization.layer_norm(x, w, b), normalization.rms_norm(x, w)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(y, x, dy, create_graph=True)
