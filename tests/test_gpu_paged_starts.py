"""Tokens in front of the first sequence belong to nobody, as those behind the last."""

import pytest
import torch

from _paged import Batch, attend, close
from mfattn.kernels import paged, rotary

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _shifted(spans, front, behind, dtype, device, hq=4, hkv=2):
    """A batch whose first ``front`` tokens are nobody's: its plan, and the batch without them."""
    b = Batch(spans, hq, hkv, 16, dtype, device, seed=front)
    starts, contexts, table = b.on_device()
    g = torch.Generator(device=device).manual_seed(front)
    n = front + b.tokens + behind
    q = torch.randn(n, hq, 64, generator=g, device=device).to(dtype)
    q[front:front + b.tokens] = b.q
    plan = paged.plan(starts + front, contexts, table, b.key_pages, tokens=n, query_heads=hq)
    return b, q, plan


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("front, behind", [(3, 0), (1, 2), (70, 5), (300, 300)])
@pytest.mark.parametrize("spans", [[(2, 9), (4, 30)], [(1, 5000)], [(90, 400), (1, 333)], [(0, 7), (3, 2)]])
def test_rows_in_front_of_the_first_sequence_are_zero(spans, front, behind, dtype, device):
    b, q, plan = _shifted(spans, front, behind, dtype, device)
    # what the allocator gives out next is not zero
    junk = torch.full(q.shape, float("nan"), dtype=dtype, device=device)
    del junk
    out = paged.attention(q, b.key_pages, b.value_pages, plan)
    end = front + b.tokens
    assert not out[:front].any() and not out[end:].any()
    close(out[front:end], *attend(b, b.q, b.key_pages, b.value_pages), "behind the front")
    given = torch.full_like(q, 5.0)
    paged.attention(q, b.key_pages, b.value_pages, plan, out=given)
    assert (given[:front] == 5).all() and (given[end:] == 5).all()
    assert torch.equal(given[front:end], out[front:end])


def test_tokens_in_front_have_no_page(device):
    b, q, plan = _shifted([(2, 9), (4, 30)], 3, 2, BF, device)
    k = torch.randn(11, 2, 64, device=device).to(BF)
    before = b.value_pages.clone()
    paged.append(k, k, b.key_pages, b.value_pages, plan, query=q, rotary=rotary.Rotary(64))
    rec = plan.token_records().cpu()
    assert (rec[:3, 1] == -1).all() and (rec[9:, 1] == -1).all() and (rec[3:9, 1] >= 0).all()
    changed = (b.value_pages != before).any(-1).any(-1).sum().item()
    assert changed == 6


def test_a_batch_of_nobodys_tokens(device):
    """Every sequence without new tokens, in the middle of a batch."""
    b = Batch([(2, 9), (4, 30)], 4, 2, 16, BF, device)
    _, contexts, table = b.on_device()
    starts = torch.tensor([4, 4, 4], dtype=torch.int32, device=device)
    plan = paged.plan(starts, contexts, table, b.key_pages, tokens=6, query_heads=4)
    junk = torch.full(b.q.shape, float("nan"), dtype=BF, device=device)
    del junk
    assert not paged.attention(b.q, b.key_pages, b.value_pages, plan).any()
