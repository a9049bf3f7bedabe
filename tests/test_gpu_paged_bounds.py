"""Steps whose tiles are cut as often as they can be: partial rows and join records at their bounds."""

import numpy as np
import pytest
import torch

from _helpers import say
from _paged import Batch
from mfattn.kernels import paged
from test_gpu_paged_nonfinite import softmax_rows

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32

CASES = [
    # spans, query heads, key heads
    ([(12000, 12000)], 16, 8),                        # more rows than can be cut
    ([(11000, 11000), (1, 40000)], 4, 2),
    ([(256, 30000)], 1, 1),                           # one tile, an item for every share
    ([(300, 20000), (1, 20000)], 2, 2),
    ([(257, 9000)] * 40, 1, 1),                       # two tiles each
    ([(128, 4000 + 7 * i) for i in range(70)], 2, 1),  # a cut in most tiles
    ([(1, 700 + 11 * i) for i in range(600)], 32, 1),  # full tiles of few rows, a cut in most
    ([(1, 90000)], 32, 1),
    ([(16, 6000)] * 9 + [(200, 5000)] * 9, 4, 2),
]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{c[0][0][0]}of{c[0][0][1]}-{c[1]}/{c[2]}")
def test_rows_of_tiles_that_are_cut(case, dtype, device):
    spans, hq, hkv = case
    say("cut tiles", dtype, len(spans), spans[0], hq, hkv)
    if dtype is F32 and sum(n * c for n, c in spans) * hq > 1.5e8:
        spans = [(max(1, n // 8), max(1, c // 2)) for n, c in spans]
    b = Batch(spans, hq, hkv, 16, dtype, device, seed=len(spans))
    out = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    rng = np.random.default_rng(hq)
    tokens = np.unique(np.concatenate((rng.integers(0, b.tokens, 60), b.starts[:20][:len(spans)],
                                       b.starts[1:21] - 1)))
    rows = [(int(t), int(rng.integers(0, hq))) for t in tokens]
    want, bound = softmax_rows(b, b.q, b.key_pages, b.value_pages, rows)
    got = torch.stack([out[t, h] for t, h in rows]).double().cpu()
    assert ((got - want).abs() - bound).max().item() <= 0
    assert bool(torch.isfinite(out).all())
