"""Paged plan, append and attention against their definitions in float64."""

import numpy as np
import pytest
import torch

from _helpers import say
from _paged import Batch, attend, close, turned
from mfattn import ops
from mfattn.kernels import attention, paged, rotary

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


# ---------------------------------------------------------------- plan


def test_plan_places_every_token(device):
    spans = [(1, 1), (0, 40), (5, 5), (3, 2), (7, 300), (0, 0), (2, 17)]
    b = Batch(spans, 4, 2, 16, BF, device, behind=3)
    rec = b.plan().token_records().cpu().numpy()
    for r, (n, context) in enumerate(spans):
        for i in range(n):
            pos, page, slot, seq = rec[b.starts[r] + i]
            assert seq == r and pos == context - n + i
            if pos >= 0:
                assert page == b.table[r, pos // 16] and slot == pos % 16
            else:
                assert page == -1
    assert (rec[b.starts[-1]:, 1] == -1).all()


def test_plan_of_many_sequences(device):
    spans = [(i % 3, 5 + i % 60) for i in range(1100)]
    b = Batch(spans, 2, 1, 8, BF, device, seed=5)
    rec = b.plan().token_records().cpu().numpy()
    want = [(c - n + i, r) for r, (n, c) in enumerate(spans) for i in range(n)]
    assert [(p, s) for p, _, _, s in rec.tolist()] == want


# ---------------------------------------------------------------- append


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["slots", "heads", "together", "apart"])
@pytest.mark.parametrize("form", ["norm+turn", "turn", "norm", "copy", "part", "odd"])
def test_append_writes_its_slots_and_nothing_else(form, layout, dtype, device):
    say("append", form, layout, dtype)
    spans = [(1, 77), (9, 9), (0, 30), (40, 100), (3, 1), (2, 130)]
    b = Batch(spans, 6, 2, 24, dtype, device, layout=layout, behind=2, spread=1.0)
    b.table[5, 5] = -1  # the page of positions 120 .. 143: given up
    b.table[4, 0] = b.key_pages.shape[0]  # no such page
    g = torch.Generator(device=device).manual_seed(1)
    qg, kg = ((1 + 0.2 * torch.randn(64, generator=g, device=device)).to(dtype) for _ in range(2))
    qg, kg = (qg, kg) if "norm" in form or form in ("part", "odd") else (None, None)
    rot = {"copy": None, "norm": None,
           "part": rotary.Rotary(64, rotary_dim=16, interleaved=True),
           "odd": rotary.Rotary(64, rotary_dim=6)}.get(form, rotary.Rotary(64, theta=1e6))
    before = b.key_pages.clone(), b.value_pages.clone()
    plan = b.plan()
    q = paged.append(b.k, b.v, b.key_pages, b.value_pages, plan, query=b.q, rotary=rot,
                     query_gain=qg, key_gain=kg, eps=1e-5)
    want_k, bound_k = before[0].double().cpu(), torch.zeros(before[0].shape, dtype=torch.float64)
    want_v = before[1].clone().cpu()
    pos = np.zeros(b.tokens, np.int64)
    for r, (n, context) in enumerate(spans):
        for i in range(n):
            t, p = b.starts[r] + i, context - n + i
            pos[t] = p
            if p < 0:
                continue
            page, slot = b.slots(r, [p])
            if page[0] >= 0:
                y, e = turned(b.k[t:t + 1], torch.tensor([p]), rot, kg)
                want_k[page[0], slot[0]], bound_k[page[0], slot[0]] = y[0], e[0]
                want_v[page[0], slot[0]] = b.v[t].cpu()
    close(b.key_pages, want_k, bound_k, "key pages")
    assert torch.equal(b.value_pages.cpu(), want_v)
    end = b.starts[-1]
    close(q[:end], *turned(b.q[:end], torch.from_numpy(pos[:end]), rot, qg), "query")


def test_append_without_queries_and_views_of_a_projection(device):
    spans = [(5, 40), (1, 9)]
    b = Batch(spans, 4, 2, 8, BF, device)
    fused = torch.randn(6, (4 + 2 + 2) * 64, device=device).to(BF)
    q, k, v = (fused[:, a * 64:z * 64].unflatten(-1, (z - a, 64)) for a, z in ((0, 4), (4, 6), (6, 8)))
    rot, plan = rotary.Rotary(64), b.plan()
    kp, vp = b.key_pages.clone(), b.value_pages.clone()
    assert paged.append(k, v, b.key_pages, b.value_pages, plan, rotary=rot) is None
    qo = paged.append(k.contiguous(), v.contiguous(), kp, vp, plan, rotary=rot, query=q)
    assert torch.equal(b.key_pages, kp) and torch.equal(b.value_pages, vp)
    # the same arithmetic as the rotation by itself
    pos = plan.token_records()[:, 0].contiguous()
    alone, ka = rotary.rotate(q, k, rot, pos)
    assert torch.equal(qo, alone)
    page, slot = plan.token_records()[:, 1].long(), plan.token_records()[:, 2].long()
    assert torch.equal(b.key_pages[page, slot], ka)


# ---------------------------------------------------------------- attention

SHAPES = [
    # spans, query heads, key heads, page size, layout
    ([(1, 1)], 2, 1, 8, "slots"),
    ([(1, 33)], 16, 8, 16, "slots"),
    ([(1, 127), (1, 128), (1, 129), (1, 4)], 16, 8, 16, "heads"),
    ([(1, 5000), (1, 0), (0, 77), (1, 63)], 8, 2, 32, "together"),
    ([(2, 2), (4, 31), (8, 40), (3, 700)], 12, 4, 24, "slots"),
    ([(16, 64), (17, 64), (16, 16), (15, 300)], 2, 1, 8, "slots"),       # 30 to 34 rows
    ([(64, 64), (65, 65), (63, 200), (1, 2)], 4, 2, 40, "heads"),        # around one tile
    ([(200, 1000), (1, 1500), (130, 130)], 8, 8, 128, "slots"),
    ([(33, 2000), (300, 301)], 3, 1, 16, "together"),
    ([(5, 3), (40, 7), (1, 0), (9, 0)], 4, 2, 8, "slots"),               # positions below zero
    ([(1, 900), (3, 60)], 40, 1, 16, "slots"),                           # 40 heads a group
    ([(2, 90)], 5, 5, 48, "heads"),
    ([(1, 20000)], 4, 4, 64, "heads"),                                   # many items
    ([(70, 3000)] * 3 + [(1, 2500)] * 20, 8, 4, 16, "slots"),            # both paths, split
    ([(90, 400), (1, 333), (2, 60)], 8, 4, 16, "apart"),                 # strides of their own
    ([(90, 400), (1, 333), (2, 60)], 9, 3, 24, "apart"),
    ([(1, 3000)] * 300, 2, 2, 16, "slots"),                              # more tiles than a round
    ([(20, 90)] * 290 + [(40, 50)], 2, 1, 8, "heads"),
]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{len(s[0])}x{s[0][0][0]}of{s[0][0][1]}-{s[1]}/{s[2]}p{s[3]}")
def test_attention(shape, dtype, device):
    spans, hq, hkv, ps, layout = shape
    say("paged attention", dtype, shape)
    b = Batch(spans, hq, hkv, ps, dtype, device, layout=layout, seed=len(spans) + ps, behind=2)
    out = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    want, bound = attend(b, b.q, b.key_pages, b.value_pages)
    close(out, want, bound, "out")
    assert not out[b.starts[-1]:].any()
    again = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n", [1, 40, 150])
def test_every_boundary_key_counts(n, dtype, device):
    """Keys at page, block, unit and item borders, and each query's own, carry the weight."""
    context = 2600
    b = Batch([(n, context)], 2, 1, 24, dtype, device, seed=n, spread=1.0)
    q = b.q.clone()
    ones = torch.zeros(64, device=device)
    ones[:] = 1.0
    q[:] = (ones * 2).to(dtype)
    marks = [0, 7, 8, 23, 24, 31, 32, 63, 64, 127, 128, 511, 512, 1279, 1280, 2559, 2560,
             context - n, context - 1]
    page, slot = b.slots(0, marks)
    # scores of 16 (+ noise) at the marked keys, of the noise elsewhere
    b.key_pages[page, slot] = (ones * 1.0).to(dtype)
    out = paged.attention(q, b.key_pages, b.value_pages, b.plan())
    want, bound = attend(b, q, b.key_pages, b.value_pages)
    close(out, want, bound, "marked keys")
    # each carries a visible share: dropping it from the definition leaves the bound
    for m in marks[:-1]:
        kp = b.key_pages.clone()
        pg, sl = b.slots(0, [m])
        kp[pg, sl] = (ones * -1.0).to(dtype)
        less, _ = attend(b, q[-1:].expand(n, 2, 64), kp, b.value_pages) if n == 1 else (None, None)
        if less is not None:
            assert ((less - want).abs() - 2 * bound).max() > 0, m


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf")])
def test_what_no_query_sees_does_not_count(junk, dtype, device):
    spans = [(1, 45), (3, 100), (80, 333), (0, 16), (1, 0)]
    b = Batch(spans, 4, 2, 16, dtype, device, spare=4)
    used = np.zeros((b.key_pages.shape[0], 16), bool)
    for r, (_, c) in enumerate(spans):
        page, slot = b.slots(r, np.arange(c)) if c else ([], [])
        used[page, slot] = True
    used[:, :][b.table[3][b.table[3] >= 0]] = False  # nobody asks the sequence without queries
    clean = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    free = torch.from_numpy(~used).to(device)
    b.key_pages[free] = junk
    b.value_pages[free] = junk
    out = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    assert torch.equal(out, clean)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["value", "key"])
def test_a_later_token_does_not_reach_an_earlier_one(where, junk, dtype, device):
    """New tokens with an infinity or NaN: earlier ones of their chunk are as without it."""
    spans = [(6, 40), (100, 300), (3, 3), (260, 400)]
    b = Batch(spans, 4, 2, 16, dtype, device, spread=1.0)
    clean = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    pages = b.value_pages if where == "value" else b.key_pages
    hit = []  # (sequence's first token, its new tokens, the new token that is hit)
    for r, i in ((0, 4), (1, 37), (1, 90), (2, 2), (3, 130)):
        n, context = spans[r]
        page, slot = b.slots(r, [context - n + i])
        pages[page, slot, 1, 5] = junk  # one dim of the second key head
        hit.append((int(b.starts[r]), n, i))
    out = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    sees = torch.zeros(b.tokens, dtype=torch.bool, device=device)
    for start, n, i in hit:
        sees[start + i:start + n] = True
    assert torch.equal(out[~sees], clean[~sees])
    assert torch.equal(out[:, :2], clean[:, :2])  # the other key head's queries
    if where == "value":
        dims = torch.arange(64, device=device) != 5
        assert torch.equal(out[sees][:, 2:][..., dims], clean[sees][:, 2:][..., dims])
        wild = out[sees][:, 2:, 5]
        assert bool(torch.isnan(wild).all() if junk != junk else (wild == junk).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads, layout", [((3, 3), "apart"), ((5, 1), "slots"), ((6, 2), "heads")])
def test_a_later_value_through_other_layouts_and_splits(heads, layout, dtype, device):
    """The same with odd numbers of key heads, and strides and a context that split its keys."""
    hq, hkv = heads
    n, context, i = 150, 6000, 61
    b = Batch([(n, context), (4, 900)], hq, hkv, 24, dtype, device, spread=1.0, layout=layout)
    clean = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    for r, at in ((0, context - n + i), (1, 898)):
        page, slot = b.slots(r, [at])
        b.value_pages[page, slot, hkv - 1, 63] = float("inf")
    out = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    sees = torch.zeros(b.tokens, dtype=torch.bool, device=device)
    sees[i:n] = sees[n + 2:] = True
    group = hq // hkv
    assert torch.equal(out[~sees], clean[~sees])
    assert torch.equal(out[:, :hq - group], clean[:, :hq - group])
    assert torch.equal(out[sees][..., :63], clean[sees][..., :63])
    assert bool((out[sees][:, hq - group:, 63] == float("inf")).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_pages_outside_the_pool_hold_no_keys(dtype, device):
    spans = [(1, 200), (2, 180), (90, 400), (1, 16), (50, 50)]
    b = Batch(spans, 4, 2, 16, dtype, device)
    b.table[0, :6] = -1                             # an evicted prefix
    b.table[1, 3] = b.key_pages.shape[0]            # one past the pool
    b.table[2, 10:14] = 2 ** 31 - 1
    b.table[3, 0] = -2 ** 31                        # nothing left
    b.table[4, 1] = -7
    out = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    want, bound = attend(b, b.q, b.key_pages, b.value_pages)
    close(out, want, bound, "pages")
    assert not out[b.starts[3]].any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_positions_beyond_the_table(dtype, device):
    """New tokens that the table has no place for are not written and see all that is there."""
    b = Batch([(2, 64), (70, 100), (3, 7)], 4, 2, 16, dtype, device)
    b.table = np.ascontiguousarray(b.table[:, :5])  # 80 slots
    b.width, b.spans = 5, [(2, 64), (70, 100), (3, 2 ** 31 - 1)]
    b.contexts = np.array([c for _, c in b.spans], np.int32)
    plan = b.plan()
    want, bound = attend(b, b.q, b.key_pages, b.value_pages)
    close(paged.attention(b.q, b.key_pages, b.value_pages, plan), want, bound, "beyond")
    rec = plan.token_records().cpu()
    assert rec[:, 0].tolist() == [62, 63, *range(30, 100), *range(2 ** 31 - 4, 2 ** 31 - 1)]
    assert (rec[2:52, 1] >= 0).all() and (rec[52:, 1] == -1).all()
    before = b.key_pages.clone()
    paged.append(b.k, b.v, b.key_pages, b.value_pages, plan)
    for r, n in ((0, 62), (1, 30), (2, 7)):  # what was cached before, and the third's page
        page, slot = b.slots(r, np.arange(n))
        assert torch.equal(b.key_pages[page, slot], before[page, slot])
    page, slot = b.slots(1, np.arange(30, 80))
    assert torch.equal(b.key_pages[page, slot], b.k[2:52])


def test_rows_behind_the_last_sequence(device):
    b = Batch([(3, 20), (40, 50)], 4, 2, 16, BF, device, behind=70)
    out = torch.full_like(b.q, 7.0)
    got = paged.attention(b.q, b.key_pages, b.value_pages, b.plan(), out=out)
    assert got is out and (out[43:] == 7).all()
    fresh = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    assert not fresh[43:].any() and torch.equal(fresh[:43], out[:43])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("first", [True, False])
def test_many_sequences_without_keys(first, dtype, device):
    """A batch filled up with sequences that have a token and no context: zeros, and the others
    as by themselves (their keys are shared out among other workgroups, so not to the bit)."""
    real, pad = [(1, 700), (40, 90), (3, 5000)], [(1, 0)] * 500 + [(200, 0)]
    b = Batch(pad + real if first else real + pad, 8, 4, 16, dtype, device)
    out = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    want, bound = attend(b, b.q, b.key_pages, b.value_pages)
    close(out, want, bound, "padded")
    none = slice(0, 700) if first else slice(44, 744)
    assert not out[none].any()


def test_shared_pages_and_strided_operands(device):
    # two sequences with a common prefix: the same pages in both rows
    b = Batch([(1, 100), (1, 110)], 16, 8, 16, BF, device)
    b.table[1, :5] = b.table[0, :5]
    fused = torch.randn(2, 32 * 64, device=device).to(BF)
    q = fused[:, 8 * 64:24 * 64].unflatten(-1, (16, 64))
    starts, contexts, _ = b.on_device()
    wide = torch.full((2, 30), -1, dtype=torch.int32, device=device)
    wide[:, 4:4 + b.width] = torch.from_numpy(b.table).to(device)
    plan = paged.plan(starts, contexts, wide[:, 4:4 + b.width], b.key_pages, tokens=2, query_heads=16)
    out = paged.attention(q, b.key_pages, b.value_pages, plan, scale=0.2)
    want, bound = attend(b, q, b.key_pages, b.value_pages, 0.2)
    close(out, want, bound, "shared")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_contiguous_cache_as_pages(dtype, device):
    g = torch.Generator(device=device).manual_seed(4)
    rows, cap = 5, 640
    kc, vc = (torch.randn(rows, cap, 2, 64, generator=g, device=device).to(dtype) for _ in range(2))
    q = torch.randn(rows, 1, 8, 64, generator=g, device=device).to(dtype)
    lengths = torch.tensor([1, 640, 333, 128, 65], dtype=torch.int32, device=device)
    kp, table = paged.cache_pages(kc, 32)
    vp, _ = paged.cache_pages(vc, 32)
    assert kp.data_ptr() == kc.data_ptr()
    starts = torch.arange(rows + 1, dtype=torch.int32, device=device)
    plan = paged.plan(starts, lengths, table, kp, tokens=rows, query_heads=8)
    out = paged.attention(q[:, 0], kp, vp, plan)
    whole = attention.cached_attention(q, kc, vc, lengths, backend="hip")[:, 0]
    # two evaluations of one definition: each within its own bound
    b = Batch([(1, int(n)) for n in lengths.tolist()], 8, 2, 32, dtype, "cpu")
    b.table, b.width, b.key_pages = table.cpu().numpy(), table.shape[1], kp
    want, bound = attend(b, q[:, 0], kp, vp)
    close(out, want, bound, "paged")
    close(whole, want, bound, "contiguous")


def test_pool_beyond_four_gigabytes(device):
    """Pages whose byte offsets pass 32 bits, in both pools."""
    pages, ps = 45000, 128  # 5.9 GB of bf16 with 8 heads
    kp = torch.empty(pages, ps, 8, 64, dtype=BF, device=device)
    vp = torch.empty_like(kp)
    ids = torch.tensor([[44999, 3, 40000, 33000], [44998, 44997, 1, 36000]], dtype=torch.int32)
    for x in ids.flatten().tolist():
        kp[x].normal_()
        vp[x].normal_()
    spans = [(1, 400), (100, 500)]
    b = Batch(spans, 16, 8, ps, BF, device, spare=1)
    b.table, b.width = ids.numpy(), 4
    starts, contexts, table = b.on_device()
    plan = paged.plan(starts, contexts, table, kp, tokens=101, query_heads=16)
    q = paged.append(b.k, b.v, kp, vp, plan, query=b.q, rotary=rotary.Rotary(64))
    page, slot = (plan.token_records()[:, i].long() for i in (1, 2))
    assert torch.equal(vp[page, slot], b.v)
    out = paged.attention(q, kp, vp, plan)
    small = torch.unique(ids.flatten()).tolist()
    b.table = np.searchsorted(small, ids.numpy()).astype(np.int32)
    ks, vs = kp[small], vp[small]
    b.key_pages, b.value_pages = ks, vs
    want, bound = attend(b, q, ks, vs)
    close(out, want, bound, "far pages")


def test_wide_spread_of_scores(device):
    """Scores from -3000 to 3000: the first key far below zero, the maximum anywhere."""
    b = Batch([(1, 700), (60, 260)], 4, 2, 16, F32, device, spread=1.0)
    q = b.q * 400
    out = paged.attention(q, b.key_pages, b.value_pages, b.plan())
    want, bound = attend(b, q, b.key_pages, b.value_pages)
    close(out, want, bound, "fp32")
    h = Batch([(1, 700), (60, 260)], 4, 2, 16, BF, device, spread=1.0)
    q = h.q * 400
    out = paged.attention(q, h.key_pages, h.value_pages, h.plan())
    want, bound = attend(h, q, h.key_pages, h.value_pages)
    close(out, want, bound, "bf16")


# ---------------------------------------------------------------- streams and graphs


def test_two_streams_share_a_plan(device):
    b = Batch([(1, 3000), (50, 900), (1, 10)], 8, 4, 16, BF, device)
    plan = b.plan()
    want = paged.attention(b.q, b.key_pages, b.value_pages, plan)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append([paged.attention(b.q, b.key_pages, b.value_pages, plan) for _ in range(5)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for group in outs for o in group)


def test_a_plan_outlives_its_last_use_on_another_stream(device):
    """A plan that is let go while another stream still reads it is not overwritten."""
    b = Batch([(1, 3000), (50, 900), (1, 10)], 8, 4, 16, BF, device)
    want = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    starts, contexts, table = b.on_device()
    table = table.long()  # the plan makes an int32 copy that only it holds
    big = torch.randn(2048, 2048, device=device)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    plan = paged.plan(starts, contexts, table, b.key_pages, tokens=b.tokens, query_heads=8)
    size = plan.buf.numel()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(40):
            big = big @ big * 1e-3  # work before the attention on its stream
        out = paged.attention(b.q, b.key_pages, b.value_pages, plan)
    shape = plan.page_table.shape
    del plan
    junk = [torch.full((size,), 255, dtype=torch.uint8, device=device) for _ in range(4)]
    tables = [torch.full(shape, -1, dtype=torch.int32, device=device) for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(out, want) and junk and tables


def test_layers_captured_over_an_eager_plan(device):
    """A graph of several layers that read one plan made outside, replayed with new queries."""
    b = Batch([(1, 500), (30, 200), (4, 40)], 8, 4, 16, BF, device)
    plan = b.plan()
    paged.attention(b.q, b.key_pages, b.value_pages, plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x = b.q
        for _ in range(3):
            x = paged.attention(x, b.key_pages, b.value_pages, plan)
    for i in range(3):
        b.q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        y = b.q
        for _ in range(3):
            y = paged.attention(y, b.key_pages, b.value_pages, plan)
        assert torch.equal(x, y), i


def test_a_misaligned_query_is_read(device):
    b = Batch([(1, 300), (40, 90)], 4, 2, 16, BF, device)
    base = torch.zeros(b.q.numel() + 1, dtype=BF, device=device)
    q = base[1:].view(b.q.shape)
    q.copy_(b.q)
    want = paged.attention(b.q, b.key_pages, b.value_pages, b.plan())
    assert q.data_ptr() % 16 and torch.equal(
        paged.attention(q, b.key_pages, b.value_pages, b.plan()), want)


def test_starts_in_disorder_stay_in_bounds(device):
    """What comes out is not defined; that the calls end and write only their rows is."""
    b = Batch([(20, 90)] * 6, 4, 2, 16, BF, device)
    _, contexts, table = b.on_device()
    n = b.tokens
    for starts in ([0, n, 0, n, 0, n, 0], [n, 90, 60, 50, 20, 10, 0], [-5, 1 << 30, -(1 << 30), 7, n, 3, n],
                   [0, 0, 0, 0, 0, 0, 0], [n] * 7):
        plan = paged.plan(torch.tensor(starts, dtype=torch.int32, device=device), contexts, table,
                          b.key_pages, tokens=n, query_heads=4)
        guard = torch.full((n + 64, 4, 64), 3.0, device=device).to(BF)
        paged.attention(b.q, b.key_pages, b.value_pages, plan, out=guard[:n])
        torch.cuda.synchronize()
        assert bool((guard[n:] == 3).all())


def test_replayed_steps(device):
    """A captured step (plan, append, attention) replayed as its sequences grow."""
    b = Batch([(1, 60), (1, 300), (3, 20)], 8, 4, 16, BF, device, width=30, spare=70)
    free = iter(sorted(set(range(b.key_pages.shape[0])) - set(b.table.flatten().tolist())))
    for r in range(3):
        for c in range(30):
            if b.table[r, c] < 0 and (c + 1) * 16 < b.contexts[r] + 64:
                b.table[r, c] = next(free)
    starts, contexts, table = b.on_device()
    rot = rotary.Rotary(64)
    gain = torch.ones(64, device=device, dtype=BF)

    def step(kp, vp):
        plan = paged.plan(starts, contexts, table, kp, tokens=b.tokens, query_heads=8)
        q = paged.append(b.k, b.v, kp, vp, plan, query=b.q, rotary=rot, query_gain=gain, key_gain=gain)
        return paged.attention(q, kp, vp, plan)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(b.key_pages.clone(), b.value_pages.clone())
    torch.cuda.current_stream().wait_stream(side)
    kp, vp = b.key_pages.clone(), b.value_pages.clone()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(kp, vp)
    with torch.cuda.graph(other):  # a second graph of the same step
        out2 = step(kp, vp)
    kp.copy_(b.key_pages)
    vp.copy_(b.value_pages)
    for i in range(4):
        contexts.add_(torch.tensor([1, 1, 3], dtype=torch.int32, device=device))
        for x in (b.q, b.k, b.v):
            x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        first = out.clone()
        want = step(b.key_pages, b.value_pages)
        other.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, want) and torch.equal(out2, want), i
        assert torch.equal(kp, b.key_pages) and torch.equal(vp, b.value_pages)


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("dtype", [F32, BF])
def test_prompt_in_chunks_then_tokens_equals_packed_attention(dtype, device):
    """A sequence that arrives in chunks and then token by token through the pages has the
    attention of the packed causal kernel over the whole (the training path), rotation included."""
    g = torch.Generator(device=device).manual_seed(11)
    total, hq, hkv = 210, 4, 2
    rot = rotary.Rotary(64, theta=1e4, rotary_dim=32, scaling="linear", factor=2.0)
    q = torch.randn(1, total, hq, 64, generator=g, device=device).to(dtype)
    k, v = (torch.randn(1, total, hkv, 64, generator=g, device=device).to(dtype) for _ in range(2))
    seg = torch.ones(1, total, dtype=torch.int32, device=device)
    qr, kr = rotary.rotate(q, k, rot)
    whole = attention.packed_causal_attention(qr, kr, v, seg, seg, backend="hip")[0]
    kp = torch.full((20, 16, hkv, 64), float("nan"), device=device).to(dtype)
    vp = kp.clone()
    table = torch.randperm(20, generator=torch.Generator().manual_seed(2))[:14].to(torch.int32)[None].to(device)
    outs, at = [], 0
    for n in [100, 57, 3, 1, 1, 40, 1, 7]:
        plan = paged.plan(torch.tensor([0, n], device=device), torch.tensor([at + n], device=device),
                          table, kp, tokens=n, query_heads=hq)
        s = slice(at, at + n)
        x = paged.append(k[0, s], v[0, s], kp, vp, plan, query=q[0, s], rotary=rot)
        assert torch.equal(x, qr[0, s])  # one rotation, whoever makes it
        outs.append(paged.attention(x, kp, vp, plan))
        at += n
    assert at == total
    b = Batch([(total, total)], hq, hkv, 16, dtype, "cpu", spare=6)
    b.table, b.width = table.cpu().numpy(), 14
    want, bound = attend(b, qr[0], kp, vp)
    close(torch.cat(outs), want, bound, "paged")
    close(whole, want, bound, "packed")


def test_plans_are_not_kept(device):
    """A plan depends on what its tensors hold when it is made."""
    b = Batch([(1, 50)], 2, 1, 16, BF, device)
    starts, contexts, table = b.on_device()
    first = paged.attention(b.q, b.key_pages, b.value_pages,
                            paged.plan(starts, contexts, table, b.key_pages, tokens=1, query_heads=2))
    contexts.fill_(20)
    second = paged.attention(b.q, b.key_pages, b.value_pages,
                             paged.plan(starts, contexts, table, b.key_pages, tokens=1, query_heads=2))
    assert not torch.equal(first, second)
    assert ops.PLANS is not None
