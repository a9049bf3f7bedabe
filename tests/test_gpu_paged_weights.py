"""bf16 attention of few rows per key head: the output's rounding is the only one that counts."""

import pytest
import torch

from _helpers import say
from _paged import Batch
from mfattn.kernels import paged
from test_gpu_paged_nonfinite import softmax_rows

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.mark.parametrize("heads, layout", [((16, 8), "slots"), ((12, 4), "heads"), ((5, 1), "slots"),
                                           ((9, 3), "apart"), ((4, 4), "together")])
@pytest.mark.parametrize("spans", [[(1, 50), (1, 700), (2, 3000)], [(1, 30000)], [(3, 900), (1, 6000), (6, 6)]])
def test_weights_of_few_rows_have_two_parts(spans, heads, layout, device):
    """Weights go into the second product as two bf16 numbers: the first is off by 2^-8 of a
    weight at most, the second holds that and is off by 2^-8 of it.  The sum adds the weights in
    float32.  Wide sums of values of either sign: outputs are far smaller than what is added."""
    say("two parts", spans, heads, layout)
    hq, hkv = heads
    b = Batch(spans, hq, hkv, 24, BF, device, layout=layout, seed=hq, spread=1.0)
    out = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    rows = [(t, h) for t in range(b.tokens) for h in range(hq)]
    want, bound = softmax_rows(b, b.q, b.key_pages, b.value_pages, rows, weights=2.0 ** -16)
    got = torch.stack([out[t, h] for t, h in rows]).double().cpu()
    assert ((got - want).abs() - bound).max().item() <= 0
