"""Infinities and NaN that a query of the paged attention does see: what a softmax over them is."""

import math

import numpy as np
import pytest
import torch

from _helpers import say
from _paged import EPS24, HALF_STEP, Batch, attend
from mfattn.kernels import attention, paged

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")

# few rows, drafts, both row blocks of a wave, many rows, contexts that split their keys, a
# sequence without keys, and rows in front of their sequence's first key
SPANS = [(1, 45), (6, 40), (100, 300), (1, 6000), (150, 3000), (1, 0), (5, 3), (33, 900)]


def softmax_rows(b, q, key_pages, value_pages, rows, scale=0.125, weights=2 * HALF_STEP[BF]):
    """(out, bound) of rows (token, head) in float64, by the definition: NaN where a visible score
    is NaN or +inf or all are -inf; a score of -inf has no weight; zeros without a key.

    The bound is that of ``_paged.attend``, over the keys that have a weight; ``weights`` is what
    rounding them to bf16 may change."""
    out = torch.zeros(len(rows), 64, dtype=torch.float64)
    bound = torch.zeros_like(out)
    group = b.hq // b.hkv
    pool_k, pool_v, q64 = key_pages.cpu(), value_pages.cpu(), q.double().cpu()
    for x, (t, h) in enumerate(rows):
        r = int(np.searchsorted(b.starts, t, side="right")) - 1
        n, context = b.spans[r]
        pos = np.arange(max(0, context - n + (t - int(b.starts[r])) + 1))
        if not len(pos):
            continue
        page, slot = b.slots(r, pos)
        page, slot = page[page >= 0], slot[page >= 0]
        if not len(page):
            continue
        k = pool_k[page, slot, h // group].double()
        v = pool_v[page, slot, h // group].double()
        s = (k @ q64[t, h]) * scale
        if bool(torch.isnan(s).any() or (s == INF).any() or (s == -INF).all()):
            out[x] = NAN
            continue
        w = s > -INF
        p = torch.softmax(s[w], 0)
        mag = ((k[w].abs() @ q64[t, h].abs()) * scale).max().item()
        out[x] = p @ v[w]
        rel = (2 * 65 * mag + 8 + int(w.sum())) * EPS24
        if b.dtype is BF:
            rel += weights
        bound[x] = rel * (p @ v[w].abs()) + HALF_STEP[b.dtype] * out[x].abs()
    return out, bound


def check(b, got, q, kp, vp, rows):
    want, bound = softmax_rows(b, q, kp, vp, rows)
    got = torch.stack([got[t, h] for t, h in rows]).double().cpu()
    nan = torch.isnan(want)
    wrong = (torch.isnan(got) != nan).any(-1).nonzero().flatten().tolist()
    assert not wrong, [rows[i] for i in wrong][:10]
    over = ((got - want).abs() - bound)[~nan]
    assert bool(torch.isfinite(got[~nan]).all()) and (not over.numel() or over.max().item() <= 0)
    return int(nan.all(-1).sum())


def some_rows(b, seed):
    """Rows of every sequence: the first, the last and a few between, all heads."""
    rng = np.random.default_rng(seed)
    rows = []
    for r, (n, _) in enumerate(b.spans):
        at = {0, n - 1, *rng.integers(0, n, size=min(n, 6)).tolist()}
        rows += [(int(b.starts[r]) + i, h) for i in sorted(at) for h in range(b.hq)]
    return rows


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("junk", [NAN, INF, -INF])
@pytest.mark.parametrize("heads, layout", [((4, 2), "slots"), ((3, 1), "heads"), ((9, 3), "apart")])
def test_rows_that_see_a_wild_key(heads, layout, junk, dtype, device):
    """One dim of one key: NaN for all that see it, an infinity by the sign of the query."""
    say("wild key", heads, layout, junk, dtype)
    hq, hkv = heads
    b = Batch(SPANS, hq, hkv, 16, dtype, device, spread=1.0, layout=layout, seed=7)
    clean = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    # (sequence, position): in the middle of a context, in the new tokens, at the far end
    for r, p in ((0, 11), (1, 37), (2, 250), (3, 4321), (4, 2900), (6, 1), (7, 880)):
        page, slot = b.slots(r, [p])
        b.key_pages[page, slot, hkv - 1, 5] = junk
    out = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    rows = some_rows(b, 1) + [(int(b.starts[2]) + i, hq - 1) for i in range(45, 56)]
    broken = check(b, out, b.q, b.key_pages, b.value_pages, rows)
    assert broken > (8 if junk == junk else 16)
    others = hq - hq // hkv  # queries of the other key heads
    assert torch.equal(out[:, :others], clean[:, :others])
    assert not out[int(b.starts[5])].any()
    again = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    assert torch.equal(out.nan_to_num(7.0), again.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("junk", [NAN, INF, -INF])
def test_a_wild_query_is_its_rows_own(junk, dtype, device):
    b = Batch(SPANS, 4, 2, 24, dtype, device, spread=1.0, seed=3)
    clean = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    q = b.q.clone()
    hit = [(int(b.starts[r]) + i, h) for r, i, h in
           ((0, 0, 1), (1, 2, 3), (2, 0, 0), (2, 64, 2), (3, 0, 0), (4, 149, 1), (4, 70, 3), (5, 0, 2),
            (6, 0, 0), (6, 4, 1), (7, 32, 2))]
    for t, h in hit:
        q[t, h, 9] = junk
    out = paged.attention(q, b.key_pages, b.value_pages, b.plan())
    broken = check(b, out, q, b.key_pages, b.value_pages, hit)
    # a row without keys stays zero, the others have a key of either sign in that dim
    no_keys = [(int(b.starts[5]), 2), (int(b.starts[6]), 0)]
    assert broken == len(hit) - len(no_keys) if junk != junk else broken >= 6
    assert not any(out[t, h].any() for t, h in no_keys)
    rest = torch.ones(out.shape[:2], dtype=torch.bool, device=device)
    for t, h in hit:
        rest[t, h] = False
    assert torch.equal(out[rest], clean[rest])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("junk", [NAN, -INF])
def test_nothing_but_wild_scores(junk, dtype, device):
    """Every key that a row sees is NaN, or has a score of -inf: no maximum rises, and the row is
    NaN all the same; rows that see another key too are finite behind -inf and NaN behind NaN."""
    spans = [(1, 30), (4, 20), (90, 200), (1, 4000), (130, 2600), (3, 2)]
    b = Batch(spans, 4, 2, 16, dtype, device, spread=1.0, seed=11)
    q = b.q.clone()
    q[..., 0] = 1.0
    b.table[4, :10] = -1          # and pages that hold no keys in front of the rest
    for r, keep in ((0, 30), (1, 18), (2, 150), (3, 4000), (4, 2500), (5, 2)):
        page, slot = b.slots(r, np.arange(keep))
        page, slot = page[page >= 0], slot[page >= 0]
        b.key_pages[page, slot, :, 0] = junk
    out = paged.attention(q, b.key_pages, b.value_pages, b.plan())
    rows = some_rows(b, 5) + [(int(b.starts[2]) + i, 0) for i in range(36, 44)]
    rows += [(int(b.starts[4]) + i, 3) for i in range(26, 34)]
    assert check(b, out, q, b.key_pages, b.value_pages, rows) > 20
    for t in (int(b.starts[5]),):  # position -1: no key
        assert not out[t].any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_given_up_pages_stay_zero_beside_wild_rows(dtype, device):
    b = Batch([(1, 100), (40, 64), (70, 3000)], 4, 2, 16, dtype, device, spread=1.0)
    b.table[0] = -1
    b.table[1] = b.key_pages.shape[0]
    b.table[2] = -1
    q = b.q.clone()
    q[::3] = NAN
    out = paged.attention(q, b.key_pages, b.value_pages, b.plan())
    assert not out.any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_nan_as_the_contiguous_decode_has_it(dtype, device):
    """Pages and a contiguous cache agree on which rows are NaN."""
    g = torch.Generator(device=device).manual_seed(4)
    rows, cap = 6, 640
    kc, vc = (torch.randn(rows, cap, 2, 64, generator=g, device=device).to(dtype) for _ in range(2))
    q = torch.randn(rows, 1, 8, 64, generator=g, device=device).to(dtype)
    lengths = torch.tensor([1, 640, 333, 128, 65, 600], dtype=torch.int32, device=device)
    kc[1, 600, 0, 3] = NAN
    kc[2, 340, 1, 3] = NAN  # behind the length
    kc[5, :600, 1, 0] = NAN
    q[4, 0, 6, 1] = NAN
    kp, table = paged.cache_pages(kc, 32)
    vp, _ = paged.cache_pages(vc, 32)
    starts = torch.arange(rows + 1, dtype=torch.int32, device=device)
    plan = paged.plan(starts, lengths, table, kp, tokens=rows, query_heads=8)
    out = paged.attention(q[:, 0], kp, vp, plan)
    whole = attention.cached_attention(q, kc, vc, lengths, backend="hip")[:, 0]
    nan = torch.zeros(rows, 8, dtype=torch.bool, device=device)
    nan[1, :4] = nan[4, 6] = nan[5, 4:] = True
    assert torch.equal(torch.isnan(out).all(-1), nan) and torch.equal(torch.isnan(out).any(-1), nan)
    assert torch.equal(torch.isnan(whole).all(-1), nan)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n", [40, 150])
def test_every_boundary_key_shows_in_the_last_row(n, dtype, device):
    """In a chunk too: a marked key that was left out would leave the last row's bound."""
    context = 2600
    b = Batch([(n, context)], 2, 1, 24, dtype, device, seed=n, spread=1.0)
    q = torch.full_like(b.q, 2.0)
    marks = [0, 7, 8, 23, 24, 31, 32, 63, 64, 127, 128, 511, 512, 1279, 1280, 2559, 2560,
             context - n, context - 1]
    page, slot = b.slots(0, marks)
    b.key_pages[page, slot] = 1.0
    out = paged.attention(q, b.key_pages, b.value_pages, b.plan())
    last = Batch([(1, context)], 2, 1, 24, dtype, device, seed=n)
    last.table = b.table
    want, bound = attend(last, q[-1:], b.key_pages, b.value_pages)
    got = out[-1:].double().cpu()
    assert ((got - want).abs() - bound).max() <= 0
    for m in marks:
        kp = b.key_pages.clone()
        pg, sl = b.slots(0, [m])
        kp[pg, sl] = -1.0
        less, _ = attend(last, q[-1:], kp, b.value_pages)
        assert ((less - want).abs() - 2 * bound).max() > 0, m
    assert math.isfinite(out.float().sum().item())
