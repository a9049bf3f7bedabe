"""Embedding lookup and its gradient against their definitions: ids, widths, vocabularies, order."""

import pytest
import torch

import _ends
from _helpers import say
from mfattn.kernels import embedding

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]


def _ids(n, v, device, seed=0, skew=True):
    g = torch.Generator(device=device).manual_seed(seed + n + v)
    u = torch.rand(n, generator=g, device=device, dtype=torch.float64)
    return (v * (u ** 4 if skew else u)).long().clamp(max=v - 1)


def _check(ids, table, scale=1.0, padding=None, seed=0):
    v, d = table.shape
    g = torch.Generator(device=table.device).manual_seed(seed + 5)
    dout = torch.randn(*ids.shape, d, generator=g, device=table.device).to(table.dtype)
    leaf = table.detach().requires_grad_()
    out = embedding.embed(ids, leaf, scale=scale, padding_id=padding)
    assert out.shape == (*ids.shape, d)
    real = (ids >= 0) & (ids < v) & (ids != (-1 if padding is None else padding))
    want = torch.where(real[..., None], table.float()[ids.long().clamp(0, v - 1)] * scale, 0)
    assert torch.equal(out, want.to(table.dtype))
    (dtable,) = torch.autograd.grad(out, leaf, dout)
    _ends.check(dtable, *_ends.embed_gradient(ids, dout, v, scale, -1 if padding is None else padding),
                "dtable")
    (again,) = torch.autograd.grad(embedding.embed(ids, leaf, scale=scale, padding_id=padding), leaf, dout)
    assert torch.equal(dtable, again)
    return dtable


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 8, 64, 127, 129, 512, 1000, 1024, 2056])
def test_widths(d, dtype, device):
    say("embed width", d, dtype)
    table = torch.randn(300, d, device=device).to(dtype)
    _check(_ids(700, 300, device), table, scale=d ** 0.5)


# chunks of 32, waves of 64, one workgroup's most, tiles of 1024 tokens and of several steps
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 65, 255, 256, 257, 1025, 8192, 8193, 9000,
                               40000, 65536, 65537, 200001])
@pytest.mark.parametrize("skew", [True, False], ids=["skewed", "even"])
def test_lengths(n, skew, device):
    say("embed length", n, skew)
    table = torch.randn(513, 72, device=device)
    _check(_ids(n, 513, device, skew=skew), table)


# one digit of the sort, its last values, two digits, three
@pytest.mark.parametrize("v", [1, 2, 255, 511, 512, 513, 4095, 65536, 262143, 262144, 300001])
def test_vocabularies(v, device):
    say("embed vocabulary", v)
    table = torch.randn(v, 16, device=device).bfloat16()
    ids = _ids(3000, v, device, skew=False)
    ids[:5] = v - 1
    _check(ids, table, scale=2.0)


@pytest.mark.parametrize("v", [30, 511, 1003, 65536, 262144])
def test_vocabularies_of_many_tokens(v, device):
    say("embed vocabulary, tiles of two steps", v)
    table = torch.randn(v, 8, device=device)
    ids = _ids(70001, v, device, skew=False)
    ids[-5:] = v - 1
    _check(ids, table, scale=0.5)


@pytest.mark.parametrize("n", [1, 32, 64, 96, 1000, 5000, 70000])
def test_one_token_over_and_over(n, device):
    table = torch.randn(1000, 136, device=device)
    _check(torch.full((n,), 7, device=device), table)
    # and two, of which one fills several chunks to their ends
    ids = torch.full((n,), 7, device=device)
    ids[: n // 3] = 8
    _check(ids, table)


@pytest.mark.parametrize("kind", [torch.int16, torch.int32, torch.int64, torch.uint8])
def test_id_types_and_shapes(kind, device):
    table = torch.randn(100, 24, device=device).bfloat16()
    ids = _ids(60, 100, device).view(3, 4, 5).to(kind)
    _check(ids, table)
    _check(ids.transpose(0, 2), table)
    _check(ids[1, 2, 3], table)


def test_ids_without_a_row(device):
    table = torch.randn(50, 40, device=device)
    ids = _ids(300, 50, device)
    ids[::7] = -1
    ids[1::11] = 50
    ids[2::13] = 1 << 40
    ids[3::17] = -(1 << 40)
    _check(ids, table)
    _check(ids, table, padding=int(ids[4]))
    _check(ids, table, padding=10 ** 15)
    none = _check(torch.full((70,), -5, device=device), table)
    assert not none.any()


def test_rows_beside_the_tokens_do_not_leak(device):
    # infinities and NaN in the gradient of padding, and in rows that no token names
    table = torch.randn(64, 32, device=device)
    table[9] = float("nan")
    ids = _ids(200, 64, device)
    ids[ids == 9] = 10
    ids[::5] = -1
    leaf = table.requires_grad_()
    out = embedding.embed(ids, leaf)
    assert out.isfinite().all()
    dout = torch.randn_like(out)
    (clean,) = torch.autograd.grad(out, leaf, dout, retain_graph=True)
    dout[::5] = float("nan")
    (same,) = torch.autograd.grad(out, leaf, dout)
    assert torch.equal(clean, same)


@pytest.mark.parametrize("how", ["rows of a wider table", "odd offset", "transposed", "expanded gradient"])
def test_views_of_any_strides(how, device):
    wide = torch.randn(90, 200, device=device).bfloat16()
    table = {"rows of a wider table": wide[:, 8:104], "odd offset": wide[:, 3:98],
             "transposed": wide[:, :90].t(), "expanded gradient": wide}[how]
    ids = _ids(500, table.shape[0], device)
    _check(ids, table)
    leaf = table.detach().requires_grad_()
    (g,) = torch.autograd.grad(embedding.embed(ids, leaf, scale=3.0).sum(), leaf)
    count = torch.bincount(ids, minlength=table.shape[0]).double()
    _ends.check(g, (3 * count)[:, None].expand(g.shape), torch.zeros(g.shape).double(), "counts")


def test_no_tokens(device):
    table = torch.randn(5, 3, device=device, requires_grad=True)
    out = embedding.embed(torch.zeros(2, 0, dtype=torch.int64, device=device), table)
    assert out.shape == (2, 0, 3)
    (g,) = torch.autograd.grad(out.sum(), table)
    assert g.shape == table.shape and not g.any()


def test_a_gradient_past_two_gigabytes(device):
    # rows of the table beyond 2^31 bytes and elements
    v, d = 2200000, 1000
    table = torch.empty(v, d, device=device, dtype=torch.bfloat16)
    ids = torch.tensor([0, v - 1, v - 2, 2147484, v - 1, 1100000], device=device)
    table[ids] = torch.randn(6, d, device=device).bfloat16()
    leaf = table.requires_grad_()
    out = embedding.embed(ids, leaf)
    assert torch.equal(out, table.detach()[ids])
    dout = torch.randn(6, d, device=device).bfloat16()
    (g,) = torch.autograd.grad(out, leaf, dout)
    assert torch.equal(g[v - 1], (dout[1].float() + dout[4].float()).bfloat16())
    for i in (0, 2, 3, 5):
        assert torch.equal(g[ids[i]], dout[i])
    g[ids] = 0
    assert g.count_nonzero().item() == 0


def test_the_gradient_is_linear(device):
    # <dout, embed(table + h)> - <dout, embed(table)> = <dtable, h>
    ids = _ids(999, 77, device)
    table, h = torch.randn(77, 40, device=device), torch.randn(77, 40, device=device)
    leaf = table.requires_grad_()
    out = embedding.embed(ids, leaf, scale=0.5)
    dout = torch.randn_like(out)
    (g,) = torch.autograd.grad(out, leaf, dout)
    with torch.no_grad():
        moved = embedding.embed(ids, table + h, scale=0.5)
    left = (dout.double() * (moved.double() - out.detach().double())).sum()
    right = (g.double() * h.double()).sum()
    # each value of both: the sum's rounding, the product's, and the gradient's own bound
    _, bound = _ends.embed_gradient(ids, dout, 77, 0.5)
    room = 4 * _ends.E * (dout.abs().double() * (moved.abs() + out.detach().abs() + 1).double()).sum() \
        + (2 * bound.to(device) * h.abs()).sum()
    assert abs(left - right) <= room


def test_the_gradient_differentiated(device):
    # <u, dtable> is linear in dout: its gradient is the lookup of u
    ids = _ids(50, 9, device)
    ids[::4] = -1
    table, u = torch.randn(9, 20, device=device, requires_grad=True), torch.randn(9, 20, device=device)
    dout = torch.randn(50, 20, device=device, requires_grad=True)
    (g,) = torch.autograd.grad(embedding.embed(ids, table, scale=2.0), table, dout, create_graph=True)
    (back,) = torch.autograd.grad(g, dout, u, create_graph=True)
    assert torch.equal(back, embedding.embed(ids, u, scale=2.0))


@pytest.mark.parametrize("v, kind", [(1003, torch.int32), (300000, torch.int64)], ids=["few", "many"])
def test_the_most_tokens(v, kind, device):
    """Small whole numbers: their sums are exact in any order (below 2^24 in fp32)."""
    n = 1 << 24
    say("embed tokens", n, v)
    g = torch.Generator(device=device).manual_seed(3)
    ids = torch.randint(-1, v, (n,), generator=g, device=device, dtype=kind)
    ids[: n // 3] = 5  # one that fills many tiles
    table = torch.zeros(v, 2, device=device, requires_grad=True)
    dout = torch.randint(-2, 3, (n, 2), generator=g, device=device).float()
    (got,) = torch.autograd.grad(embedding.embed(ids, table), table, dout)
    got = got.double().cpu()
    # (on the host: millions of atomic additions to one 64-bit address take minutes on the GPU)
    at, d = torch.where(ids < 0, v, ids).long().cpu(), dout.double().cpu()
    want = torch.stack([torch.bincount(at, d[:, i], minlength=v + 1)[:v] for i in (0, 1)], 1)
    assert want.abs().max() < 1 << 24 and torch.equal(got, want)
    with pytest.raises(ValueError, match="at most"):
        embedding.embed(torch.cat([ids, ids[:1]]), table)
