"""Gradients of an id that very many tokens have: float32 sums whose rounding does not grow with the
tokens."""

import pytest
import torch

from _ends import E
from _helpers import say
from mfattn.kernels import embedding

pytestmark = pytest.mark.gpu


# equal values round the same way every time: the worst that a long sum meets
@pytest.mark.parametrize("value", [0.1, 1 / 3, 0.7, 1.1])
@pytest.mark.parametrize("n", [70001, 1 << 20, 3 << 20])
def test_one_id(n, value, device):
    say("embed long", n, value)
    dout = torch.full((n, 64), value, device=device)
    leaf = torch.zeros(5, 64, device=device).requires_grad_()
    (got,) = torch.autograd.grad(embedding.embed(torch.full((n,), 3, device=device), leaf), leaf, dout)
    want = n * float(dout[0, 0])
    # terms in a row: a wave's 64 tokens, 64 of their sums, those of a quarter of them, four waves'
    # and the scale
    deep = 64 + 64 + -(-n // (64 * 64 * 4)) + 4 + 1
    assert ((got[3].double() - want).abs() <= deep * E * want).all()
    assert not got[[0, 1, 2, 4]].any()


def test_a_frequent_id_among_others(device):
    n = 1 << 20
    g = torch.Generator(device=device).manual_seed(4)
    ids = torch.randint(0, 999, (n,), generator=g, device=device)
    ids[torch.rand(n, generator=g, device=device) < 0.5] = 400
    dout = 0.2 + torch.rand(n, 32, generator=g, device=device)
    leaf = torch.zeros(999, 32, device=device).requires_grad_()
    (got,) = torch.autograd.grad(embedding.embed(ids, leaf), leaf, dout)
    count = int((ids == 400).sum())
    want = dout[ids == 400].double().sum(0)
    deep = 64 + 64 + -(-count // (64 * 64 * 4)) + 1 + 4 + 1
    assert ((got[400].double() - want).abs() <= deep * E * want).all()
