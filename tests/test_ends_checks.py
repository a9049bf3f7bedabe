"""Refusals of the norms, the embedding and the distillation loss (no GPU needed)."""

import pytest
import torch
from torch.autograd import forward_ad

from mfattn import _lib
from mfattn.kernels import distillation, embedding, normalization

L = _lib.LIB
P = 1 << 20  # an address that no refused call reads


def _msg():
    return L.mf_last_error().decode()


def _norm(**kw):
    a = dict(x=P, xs=64, w=P, b=None, dt=1, pdt=1, rows=4, dim=64, center=1, eps=1e-5, y=2 * P,
             st=None)
    a.update(kw)
    return L.mf_norm(*a.values(), None)


def _norm_bwd(**kw):
    a = dict(x=P, xs=64, w=P, st=P, dy=P, dys=64, dt=1, pdt=1, rows=4, dim=64, center=1, dx=2 * P,
             dw=P, db=P, ws=P, n=1 << 30)
    a.update(kw)
    return L.mf_norm_bwd(*a.values(), None)


def _embed(**kw):
    a = dict(ids=P, size=8, t=P, ts=64, dt=1, n=4, v=10, d=64, pad=-1, scale=1.0, out=P)
    a.update(kw)
    return L.mf_embed(*a.values(), None)


def _embed_bwd(**kw):
    a = dict(ids=P, size=8, g=P, gs=64, dt=1, n=4, v=10, d=64, pad=-1, scale=1.0, out=P, ws=P,
             nb=1 << 30)
    a.update(kw)
    return L.mf_embed_bwd(*a.values(), None)


def _distill(**kw):
    a = dict(z=P, zs=100, t=P, tdt=1, ids=P, size=4, total=None, w=None, dt=1, n=4, v=100, k=8,
             temp=1.0, loss=P, st=None, nb=0, g=None, gs=0)
    a.update(kw)
    return L.mf_distill(*a.values(), None)


def _distill_bwd(**kw):
    a = dict(z=P, zs=100, ids=P, size=4, w=None, st=P, nb=1 << 20, up=P, dt=1, n=4, v=100, k=8,
             temp=1.0, g=2 * P, gs=100)
    a.update(kw)
    return L.mf_distill_bwd(*a.values(), None)


ARG, SHAPE, DTYPE, WS = (_lib.ERR_INVALID_ARGUMENT, _lib.ERR_SHAPE, _lib.ERR_DTYPE,
                         _lib.ERR_WORKSPACE)


@pytest.mark.parametrize("call, kw, code, text", [
    (_norm, dict(x=None), ARG, "non-null"),
    (_norm, dict(dt=3), DTYPE, "dtype"),
    (_norm, dict(dt=0, pdt=1), DTYPE, "float32"),
    (_norm, dict(rows=0), ARG, "positive"),
    (_norm, dict(dim=-1), ARG, "positive"),
    (_norm, dict(dim=16385, xs=16385), SHAPE, "at most"),
    (_norm, dict(rows=(1 << 22) + 1), SHAPE, "at most"),
    (_norm, dict(xs=63), SHAPE, "63 elements between rows"),
    (_norm, dict(eps=-1.0), ARG, "eps"),
    (_norm, dict(eps=float("nan")), ARG, "eps"),
    (_norm, dict(center=0, b=P), ARG, "no bias"),
    (_norm, dict(xs=65, y=P), SHAPE, "not dense"),
    (_norm_bwd, dict(st=None), ARG, "non-null"),
    (_norm_bwd, dict(dys=3), SHAPE, "dy: 3 elements"),
    (_norm_bwd, dict(dx=P), ARG, "must not be x"),
    (_norm_bwd, dict(dy=2 * P, dys=65), SHAPE, "not dense"),
    (_norm_bwd, dict(rows=1 << 20, n=8), WS, "workspace holds 8"),
    (_norm_bwd, dict(rows=1 << 20, ws=None), WS, "workspace holds 0"),
    (_norm_bwd, dict(center=0), ARG, "no bias"),
    (_norm_bwd, dict(rows=0), ARG, "positive"),
    (_embed, dict(table=None) and dict(t=None), ARG, "non-null"),
    (_embed, dict(size=2), DTYPE, "4 or 8 bytes"),
    (_embed, dict(dt=2), DTYPE, "dtype"),
    (_embed, dict(n=0), ARG, "positive"),
    (_embed, dict(n=(1 << 24) + 1), SHAPE, "at most"),
    (_embed, dict(d=(1 << 16) + 1, ts=1 << 20), SHAPE, "at most"),
    (_embed, dict(n=1 << 24, d=2048, ts=2048), SHAPE, "at most"),
    (_embed, dict(v=(1 << 27) + 1), SHAPE, "at most"),
    (_embed, dict(scale=float("inf")), ARG, "scale"),
    (_embed, dict(ts=63), SHAPE, "table: 63"),
    (_embed_bwd, dict(out=P + 8), ARG, "aligned"),
    (_embed_bwd, dict(nb=100), WS, "workspace holds 100"),
    (_embed_bwd, dict(ws=None), WS, "workspace holds 0"),
    (_embed_bwd, dict(gs=1), SHAPE, "dout: 1"),
    (_embed_bwd, dict(ids=None), ARG, "non-null"),
    (_distill, dict(z=None), ARG, "non-null"),
    (_distill, dict(tdt=5), DTYPE, "teacher dtype"),
    (_distill, dict(size=1), DTYPE, "4 or 8 bytes"),
    (_distill, dict(k=0), ARG, "positive"),
    (_distill, dict(k=1025), SHAPE, "at most"),
    (_distill, dict(v=393217, zs=393217), SHAPE, "at most"),
    (_distill, dict(n=1 << 20, v=65536, zs=65536), SHAPE, "at most"),
    (_distill, dict(n=(1 << 21) + 1), SHAPE, "at most"),
    (_distill, dict(temp=0.0), ARG, "temperature"),
    (_distill, dict(temp=float("inf")), ARG, "temperature"),
    (_distill, dict(zs=99), SHAPE, "logits: 99"),
    (_distill, dict(g=2 * P, gs=99), SHAPE, "dlogits: 99"),
    (_distill, dict(g=P, gs=120), SHAPE, "their stride"),
    (_distill, dict(st=P, nb=4 * 4 * 11), WS, "stats hold"),
    (_distill_bwd, dict(up=None), ARG, "non-null"),
    (_distill_bwd, dict(g=P), ARG, "must not be the logits"),
    (_distill_bwd, dict(nb=10), WS, "stats hold 10"),
    (_distill_bwd, dict(gs=10), SHAPE, "dlogits: 10"),
    (_distill_bwd, dict(temp=-1.0), ARG, "temperature"),
])
def test_c_refusals(call, kw, code, text):
    assert call(**kw) == code
    assert text in _msg()


def test_sizes_of_refused_calls_are_zero():
    assert L.mf_norm_bwd_workspace_bytes(0, 4, 1) == 0
    assert L.mf_norm_bwd_workspace_bytes(4, 16385, 1) == 0
    assert L.mf_norm_bwd_workspace_bytes(4, 4, 9) == 0
    assert L.mf_embed_bwd_workspace_bytes(0, 4, 1) == 0
    assert L.mf_embed_bwd_workspace_bytes(1 << 24, 4, 1 << 16) == 0
    assert L.mf_distill_stats_bytes(4, 0) == 0
    assert L.mf_distill_stats_bytes(4, 8) == 4 * 4 * 12
    assert L.mf_norm_bwd(P, 64, P, P, P, 64, 1, 1, 4, 64, 1, None, None, None, None, 0, None) == 0


def _f(*shape):
    return torch.zeros(*shape)


def _i(*shape):
    return torch.zeros(*shape, dtype=torch.int64)


@pytest.mark.parametrize("call, match", [
    (lambda: normalization.layer_norm(_f(2, 4), _f(4)), "GPU only"),
    (lambda: normalization.layer_norm(_f(2, 0), _f(0)), "D positive"),
    (lambda: normalization.layer_norm(torch.tensor(1.0), _f(1)), "D positive"),
    (lambda: normalization.layer_norm(_f(2, 4), _f(5)), r"weight must be \[4\]"),
    (lambda: normalization.layer_norm(_f(2, 4), _f(4), _f(1)), r"bias must be \[4\]"),
    (lambda: normalization.layer_norm(_f(2, 4).half(), _f(4)), "dtype"),
    (lambda: normalization.layer_norm(_f(2, 4), _f(4).bfloat16()), "weight must be"),
    (lambda: normalization.layer_norm(_f(2, 4).bfloat16(), _f(4), _f(4).bfloat16()), "share one dtype"),
    (lambda: normalization.rms_norm(_f(2, 4), _f(4), eps=float("nan")), "eps"),
    (lambda: normalization.rms_norm(_f(2, 4), _f(4), eps=-1e-9), "eps"),
    (lambda: embedding.embed(_i(3), _f(4, 2)), "GPU only"),
    (lambda: embedding.embed(_i(3), _f(4)), "table must be"),
    (lambda: embedding.embed(_i(3), _f(0, 4)), "table must be"),
    (lambda: embedding.embed(_f(3), _f(4, 2)), "integers"),
    (lambda: embedding.embed(_i(3).bool(), _f(4, 2)), "integers"),
    (lambda: embedding.embed(_i(3), _f(4, 2).double()), "dtype"),
    (lambda: embedding.embed(_i(3), _f(4, 2), scale=float("nan")), "scale"),
    (lambda: embedding.embed(_i(3), _f(4, 2), padding_id=1 << 63), "padding_id"),
    (lambda: distillation.top_logits_loss(_f(2, 9), _f(2, 3), _i(2, 3)), "GPU only"),
    (lambda: distillation.top_logits_loss(_f(2, 9), _f(2, 3), _i(2, 4)), "must be"),
    (lambda: distillation.top_logits_loss(_f(2, 9), _f(1, 3), _i(1, 3)), "must be"),
    (lambda: distillation.top_logits_loss(_f(2, 9), _f(2, 0), _i(2, 0)), "must be"),
    (lambda: distillation.top_logits_loss(_f(2, 9), _f(2, 3), _f(2, 3)), "integers"),
    (lambda: distillation.top_logits_loss(_f(2, 9).half(), _f(2, 3), _i(2, 3)), "dtype"),
    (lambda: distillation.top_logits_loss(_f(2, 9), _f(2, 3).half(), _i(2, 3)), "dtype"),
    (lambda: distillation.top_logits_loss(_f(2, 9), _f(2, 3), _i(2, 3), temperature=0), "temperature"),
    (lambda: distillation.top_logits_loss(_f(2, 9), _f(2, 3), _i(2, 3), weights=_f(3)), "weights must be"),
    (lambda: distillation.top_logits_loss(_f(2, 9), _f(2, 3), _i(2, 3), weights=_i(2)), "floating"),
    (lambda: distillation.top_logits_loss(_f(2, 9), _f(2, 3), _i(2, 3), teacher_total=_f(2, 1)),
     "teacher_total must be"),
    (lambda: distillation.top_logits_loss(_f(2, 9), _f(2, 3).requires_grad_(), _i(2, 3)), "logits alone"),
    (lambda: distillation.top_logits_loss(_f(2, 9), _f(2, 3), _i(2, 3), weights=_f(2).requires_grad_()),
     "logits alone"),
    (lambda: distillation.top_logits_loss_and_gradient(_f(2, 9).requires_grad_(), _f(2, 3), _i(2, 3)),
     "records no graph"),
])
def test_python_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def test_tangents_are_refused():
    def dual(t):
        return forward_ad.make_dual(t, torch.ones_like(t))

    with forward_ad.dual_level():
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in (lambda: normalization.layer_norm(dual(_f(2, 4)), _f(4)),
                             lambda: normalization.rms_norm(_f(2, 4), dual(_f(4))),
                             lambda: embedding.embed(_i(3), dual(_f(4, 2))),
                             lambda: distillation.top_logits_loss(dual(_f(2, 9)), _f(2, 3), _i(2, 3)),
                             lambda: distillation.top_logits_loss_and_gradient(
                                 _f(2, 9), dual(_f(2, 3)), _i(2, 3))):
                    with pytest.raises(ValueError, match="carries a tangent"):
                        call()
