"""Sums over many rows and tokens, of whole numbers: exact in float32 in any order, so that a row
that is left out or counted twice shows."""

import pytest
import torch

import _ends
from _ends import E
from _helpers import say
from mfattn.kernels import embedding, normalization

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]


def _groups(dim, dtype):
    """Groups of lanes that take rows in turn, of all workgroups of the norm's backward pass."""
    n = 8 if dtype is torch.bfloat16 else 4
    vectors = -(-dim // n)
    lanes = 16 if vectors <= 16 else 64 if vectors <= 128 else 256 if vectors <= 256 else 512
    held = -(-vectors // lanes) * n
    return 512 // lanes * (256 if held > (16 if lanes < 512 else 8) else 512)


# rows of every number of lanes, three and more in turn to each group, an odd number of them
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vectors, rows", [(8, 32771), (16, 100003), (32, 8197), (64, 20483), (128, 8193),
                                           (128, 32771), (256, 4101), (512, 2051), (1024, 1539),
                                           (2048, 1031)])
@pytest.mark.parametrize("odd", [0, 3])
def test_norm_gradients_of_many_rows(odd, vectors, rows, dtype, device):
    dim = vectors * (8 if dtype is torch.bfloat16 else 4) - odd
    say("norm rows", rows, dim, dtype)
    g = torch.Generator(device=device).manual_seed(rows + dim)
    x = torch.randn(rows, dim, generator=g, device=device).to(dtype)
    dy = torch.randint(-4, 5, (rows, dim), generator=g, device=device).to(dtype)
    w, b = (torch.randn(dim, generator=g, device=device) for _ in range(2))
    per = -(-rows // _groups(dim, dtype))
    assert per >= 3 or vectors >= 1024
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = normalization.layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(db.double(), dy.double().sum(0))
    want = _ends.norm(x.detach(), w.detach(), b.detach(), 1e-5, True, dy)
    _ends.check(y.detach(), *want["y"], "y")
    _ends.check(dx, *want["dx"], "dx")
    # dweight: a group adds `per` rows, then come lanes and waves, the partials in 16 shares, and these
    xd = x.detach().double()
    off = xd - xd.mean(-1, keepdim=True)
    h = off * ((off * off).mean(-1, keepdim=True) + 1e-5) ** -0.5
    size = (dy.double() * h).abs().sum(0)
    # what a normalised value is off by: y's bound without weight, bias and rounding
    ones = torch.ones_like(w.detach())
    h_e = _ends.norm(x.detach(), ones, None, 1e-5, True)["y"][1]
    deep = per + 2 + 8 + 512 // 16 + 16
    _ends.check(dw, (dy.double() * h).sum(0), (dy.double().abs() * h_e).sum(0) + deep * E * size, "dweight")


# around the tokens at which a wave's share doubles from 8 to 64, and the ends of the sort's paths
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [7, 8, 9, 1023, 1024, 1025, 8191, 8192, 8193, 16383, 16384, 16385, 32767, 32768,
                               32769, 65535, 65536, 65537, 131073])
@pytest.mark.parametrize("d", [5, 64, 600])
def test_embedding_gradients_of_runs_around_a_share(d, n, dtype, device):
    """Ids whose tokens end just before, at and behind the shares' ends, in any order of tokens."""
    say("embed runs", n, d, dtype)
    g = torch.Generator(device=device).manual_seed(n + d)
    lengths = [1, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 1000, 4097]
    pick = torch.randint(0, len(lengths), (n,), generator=g, device=device)
    ids = torch.repeat_interleave(torch.arange(n, device=device),
                                  torch.tensor(lengths, device=device)[pick])[:n]
    v = int(ids.max()) + 3
    ids = ids[torch.randperm(n, generator=g, device=device)]
    dout = torch.randint(-3, 4, (n, d), generator=g, device=device).to(dtype)
    leaf = torch.zeros(v, d, device=device, dtype=dtype).requires_grad_()
    (got,) = torch.autograd.grad(embedding.embed(ids, leaf), leaf, dout)
    want = torch.zeros(v, d, dtype=torch.float64).index_add_(0, ids.cpu(), dout.double().cpu())
    assert torch.equal(got.cpu(), want.to(dtype))


@pytest.mark.parametrize("n", [100, 1024, 5000, 8192, 8193, 70001, 300000, 700001])
@pytest.mark.parametrize("share", [1.0, 0.5, 0.1])
def test_embedding_gradients_of_one_frequent_id(share, n, device):
    g = torch.Generator(device=device).manual_seed(n)
    ids = torch.randint(0, 999, (n,), generator=g, device=device)
    ids[torch.rand(n, generator=g, device=device) < share] = 400
    dout = torch.randint(-3, 4, (n, 130), generator=g, device=device).float()
    leaf = torch.zeros(999, 130, device=device).requires_grad_()
    (got,) = torch.autograd.grad(embedding.embed(ids, leaf), leaf, dout)
    want = torch.zeros(999, 130, dtype=torch.float64).index_add_(0, ids.cpu(), dout.double().cpu())
    assert torch.equal(got.double().cpu(), want)
