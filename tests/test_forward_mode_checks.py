"""Operands that carry a forward-mode tangent, where a call has no derivative (no GPU needed)."""

import pytest
import torch
from torch.autograd import forward_ad

from mfattn import _lib, ops
from mfattn.kernels import paged

L = _lib.LIB


def _plan():
    n = L.mf_paged_plan_bytes(2, 4, 4, 2, _lib.DTYPE_F32)
    return paged.Plan(torch.zeros(n, dtype=torch.uint8), torch.zeros(2, 3, dtype=torch.int32), 2, 4, 4,
                      torch.Size((7, 16, 2, 64)), _lib.DTYPE_F32)


def test_a_tangent_is_seen_only_where_there_is_one():
    x = torch.ones(3)
    assert not ops.carries_tangent(x, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        assert not dual.requires_grad
        assert ops.carries_tangent(None, x, dual) and not ops.carries_tangent(x)
        with torch.no_grad():
            assert ops.carries_tangent(dual)
    assert not ops.carries_tangent(dual)


@pytest.mark.parametrize("which", ["query", "key", "value", "key_pages", "value_pages", "query_gain",
                                   "key_gain"])
@pytest.mark.parametrize("grad", [True, False])
def test_append_refuses_a_tangent(which, grad):
    args = dict(key=torch.zeros(4, 2, 64), value=torch.zeros(4, 2, 64),
                key_pages=torch.zeros(7, 16, 2, 64), value_pages=torch.zeros(7, 16, 2, 64),
                query=torch.zeros(4, 4, 64), query_gain=torch.ones(64), key_gain=torch.ones(64))
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        with pytest.raises(ValueError, match="GPU only"):
            paged.append(plan=_plan(), **args)
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(ValueError, match="carries a tangent"):
            paged.append(plan=_plan(), **args)


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("grad", [True, False])
def test_attention_refuses_a_tangent(which, grad):
    args = [torch.zeros(4, 4, 64), torch.zeros(7, 16, 2, 64), torch.zeros(7, 16, 2, 64)]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(ValueError, match="carries a tangent"):
            paged.attention(*args, _plan())
