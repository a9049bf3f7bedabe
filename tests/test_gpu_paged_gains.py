"""Gains of the append in another dtype than the pages."""

import pytest
import torch

from _paged import Batch
from mfattn.kernels import paged

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype, gain_dtype", [(BF, F32), (BF, torch.float64), (F32, BF), (F32, torch.float64)])
def test_gains_are_taken_in_the_pages_dtype(dtype, gain_dtype, device):
    b = Batch([(5, 40), (1, 9)], 4, 2, 16, dtype, device, spread=1.0)
    g = torch.Generator(device=device).manual_seed(1)
    qg, kg = ((1 + 0.3 * torch.randn(64, generator=g, device=device)).to(gain_dtype) for _ in range(2))
    pools = [(b.key_pages.clone(), b.value_pages.clone()) for _ in range(2)]
    out = [paged.append(b.k, b.v, *pool, b.plan(), query=b.q, query_gain=x, key_gain=y)
           for pool, x, y in zip(pools, (qg, qg.to(dtype)), (kg, kg.to(dtype)))]
    assert torch.equal(out[0], out[1]) and torch.equal(pools[0][0], pools[1][0])
    # every other one of a wider vector is read by its values too
    wide = torch.zeros(128, dtype=dtype, device=device)
    wide[::2] = kg.to(dtype)
    again = (b.key_pages.clone(), b.value_pages.clone())
    paged.append(b.k, b.v, *again, b.plan(), key_gain=wide[::2])
    assert torch.equal(again[0], pools[0][0])
