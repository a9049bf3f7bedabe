"""Refusals of the rotary and paged entry points, and a model's frequencies (no GPU needed).

Every refusal comes from the host before anything is enqueued: through the
Python functions with host tensors, and through the C ABI with pointers that
are never followed.
"""

import copy
import ctypes
import math
import pickle

import pytest
import torch

from mfattn import _lib
from mfattn.kernels import paged, rotary

L = _lib.LIB
PTR = ctypes.c_void_p(1 << 20)  # never followed: every call here is refused


def _msg():
    return L.mf_last_error().decode()


# ---------------------------------------------------------------- frequencies


def test_frequencies_of_every_scaling():
    base = [1e6 ** (-2 * i / 64) for i in range(32)]
    assert rotary.Rotary(64, theta=1e6).frequencies == tuple(base)
    lin = rotary.Rotary(64, theta=1e6, scaling="linear", factor=4.0)
    assert lin.frequencies == tuple(f / 4 for f in base) and lin.magnitude == 1.0
    grown = rotary.Rotary(64, theta=1e6, scaling="base", factor=4.0).frequencies
    assert grown[0] == 1.0 and math.isclose(grown[-1], base[-1] / 4, rel_tol=1e-12)
    bands = rotary.Rotary(64, theta=1e6, scaling="bands", factor=8.0, original_length=8192).frequencies
    for f, g in zip(base, bands):
        turns = 8192 * f / (2 * math.pi)
        if turns >= 4:
            assert g == f
        elif turns <= 1:
            assert math.isclose(g, f / 8, rel_tol=1e-12)
        else:
            assert f / 8 < g < f
    ramp = rotary.Rotary(64, theta=1e6, scaling="ramp", factor=8.0, original_length=8192)
    assert ramp.frequencies[0] == 1.0 and math.isclose(ramp.frequencies[-1], base[-1] / 8, rel_tol=1e-12)
    assert all(f / 8 - 1e-18 <= g <= f for f, g in zip(base, ramp.frequencies))
    assert math.isclose(ramp.magnitude, 1 + 0.1 * math.log(8.0))
    mine = rotary.Rotary(8, frequencies=[1.0, 0.5, 0.25, 0.0], magnitude=2.0)
    assert mine.frequencies == (1.0, 0.5, 0.25, 0.0) and mine.magnitude == 2.0


@pytest.mark.parametrize("kw, text", [
    (dict(head_dim=7), "head_dim must be even"),
    (dict(head_dim=0), "head_dim must be even"),
    (dict(head_dim=2048), "head_dim must be even"),
    (dict(head_dim=64, rotary_dim=3), "rotary_dim must be even"),
    (dict(head_dim=64, rotary_dim=66), "rotary_dim must be even"),
    (dict(head_dim=512), "rotary_dim must be even"),
    (dict(head_dim=64, scaling="other"), "Unsupported rotary scaling"),
    (dict(head_dim=64, theta=1.0), "theta"),
    (dict(head_dim=64, theta=float("nan")), "theta"),
    (dict(head_dim=64, scaling="linear", factor=0.5), "factor"),
    (dict(head_dim=64, scaling="bands", factor=2.0), "original_length"),
    (dict(head_dim=64, scaling="ramp", factor=2.0, original_length=100, fast=1.0, slow=2.0), "slow"),
    (dict(head_dim=64, frequencies=[1.0]), "32 numbers"),
    (dict(head_dim=4, frequencies=[1.0, float("inf")]), "finite"),
    (dict(head_dim=64, magnitude=float("nan")), "finite"),
])
def test_rotary_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        rotary.Rotary(**kw)


@pytest.mark.parametrize("q, k, text", [
    ((2, 3, 4, 32), None, "heads of 64"),
    ((3, 64), None, "query must be"),
    ((2, 3, 4, 64), (2, 4, 2, 64), "share batch"),
    ((2, 3, 4, 64), (2, 3, 2, 64), "GPU only"),
])
def test_rotate_refuses(q, k, text):
    rot = rotary.Rotary(64)
    with pytest.raises(ValueError, match=text):
        rotary.rotate(torch.zeros(q), None if k is None else torch.zeros(k), rot)
    with pytest.raises(ValueError, match="must be a Rotary"):
        rotary.rotate(torch.zeros(q), None, 1e4)


def test_rotate_refuses_dtypes():
    rot = rotary.Rotary(64)
    with pytest.raises(ValueError, match="Unsupported dtype"):
        rotary.rotate(torch.zeros(1, 2, 3, 64, dtype=torch.float16), None, rot)
    with pytest.raises(ValueError, match="share batch"):
        rotary.rotate(torch.zeros(1, 2, 3, 64), torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16), rot)


# ---------------------------------------------------------------- paged, Python


def _plan_args(**kw):
    args = dict(query_starts=torch.tensor([0, 1, 4], dtype=torch.int32),
                context_lengths=torch.tensor([5, 9], dtype=torch.int32),
                page_table=torch.zeros(2, 3, dtype=torch.int32),
                key_pages=torch.zeros(7, 16, 2, 64), tokens=4, query_heads=4)
    args.update(kw)
    return args


@pytest.mark.parametrize("kw, text", [
    (dict(query_starts=torch.zeros(2, dtype=torch.int32)), "query_starts must be"),
    (dict(context_lengths=torch.zeros(3, dtype=torch.int32)), "context_lengths must be"),
    (dict(context_lengths=torch.zeros(2)), "must hold integers"),
    (dict(page_table=torch.zeros(6, dtype=torch.int32)), "page_table must be"),
    (dict(page_table=torch.zeros(2, 3)), "must hold integers"),
    (dict(key_pages=torch.zeros(7, 16, 2, 32)), "head_dim 64"),
    (dict(key_pages=torch.zeros(7, 16, 128)), "pages must be"),
    (dict(key_pages=torch.zeros(7, 16, 2, 64, dtype=torch.float16)), "Unsupported dtype"),
    (dict(), "GPU only"),
])
def test_plan_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        paged.plan(**_plan_args(**kw))


def _host_plan(tokens=4, hq=4, pool=(7, 16, 2, 64), code=_lib.DTYPE_F32):
    n = L.mf_paged_plan_bytes(2, tokens, hq, pool[2], code)
    return paged.Plan(torch.zeros(n, dtype=torch.uint8), torch.zeros(2, 3, dtype=torch.int32), 2,
                      tokens, hq, torch.Size(pool), code)


def test_attention_refuses():
    plan, kp, q = _host_plan(), torch.zeros(7, 16, 2, 64), torch.zeros(4, 4, 64)
    graded = torch.zeros(4, 4, 64, requires_grad=True)
    for args, text in (
            ((q[:3], kp, kp), "query must be"),
            ((q[:, :2], kp, kp), "query must be"),
            ((q.bfloat16(), kp, kp), "share one dtype"),
            ((q.bfloat16(), kp.bfloat16(), kp.bfloat16()), "another dtype"),
            ((q, kp[:6], kp), "the plan is for pages"),
            ((q, kp, kp[:, :8]), "the plan is for pages"),
            ((graded, kp, kp), "no backward"),
            ((q, kp, kp), "GPU only")):
        with pytest.raises(ValueError, match=text):
            paged.attention(*args, plan)


def test_append_refuses():
    plan, kp, vp = _host_plan(), torch.zeros(7, 16, 2, 64), torch.zeros(7, 16, 2, 64)
    k, q, g = torch.zeros(4, 2, 64), torch.zeros(4, 4, 64), torch.ones(64)
    graded = torch.zeros(4, 2, 64, requires_grad=True)
    rot = rotary.Rotary(64)
    for args, kw, text in (
            ((k[:3], k, kp, vp), {}, "keys and values must be"),
            ((k, k[:, :1], kp, vp), {}, "keys and values must be"),
            ((k, k, kp, vp), dict(query=q[:, :3]), "query must be"),
            ((k, k, kp, vp), dict(query_gain=g), "needs a query"),
            ((k, k, kp, vp), dict(key_gain=g[:32]), "gains must be"),
            ((k, k, kp, vp), dict(rotary=rotary.Rotary(128)), "rotary must be"),
            ((k, k, kp, vp), dict(rotary=1e4), "rotary must be"),
            ((k, k.bfloat16(), kp, vp), {}, "share one dtype"),
            ((k, k, kp, kp), {}, "pages of their own"),
            ((k, k, kp, vp[:5]), {}, "the plan is for pages"),
            ((graded, k, kp, vp), {}, "no backward"),
            ((k, k, kp, vp), dict(query=q, rotary=rot), "GPU only")):
        with pytest.raises(ValueError, match=text):
            paged.append(*args, plan, **kw)


def test_wide_integers_keep_their_order():
    x = torch.tensor([2 ** 40, -2 ** 40, 2 ** 32, 5, -1])
    assert paged._int32(x, (5,), "x").tolist() == [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 5, -1]


def test_cache_pages_refuses():
    with pytest.raises(ValueError, match="whole pages"):
        paged.cache_pages(torch.zeros(2, 100, 2, 64), 16)
    with pytest.raises(ValueError, match="contiguous"):
        paged.cache_pages(torch.zeros(2, 64, 4, 64)[:, :, ::2], 16)
    pages, table = paged.cache_pages(torch.zeros(2, 64, 4, 64), 16)
    assert pages.shape == (8, 16, 4, 64) and table.tolist() == [[0, 1, 2, 3], [4, 5, 6, 7]]


def test_rotate_refuses_positions_that_are_no_integers():
    q = torch.zeros(1, 3, 2, 64)
    for positions in (torch.zeros(3), 1.5, torch.ones(1, 3, dtype=torch.bool), [0.0, 1.0, 2.0]):
        with pytest.raises(ValueError, match="positions must be integers"):
            rotary.rotate(q, None, rotary.Rotary(64), positions)


@pytest.mark.parametrize("again", [copy.copy, copy.deepcopy,
                                   lambda r: pickle.loads(pickle.dumps(r))])
def test_copies_have_turns_of_their_own(again):
    rot = rotary.Rotary(128, theta=5e5, rotary_dim=64, interleaved=True, scaling="ramp", factor=8.0,
                        original_length=4096)
    turns = list(rot._turns)
    new = again(rot)
    assert new._args[0] == ctypes.addressof(new._turns) != rot._args[0]
    assert list(new._turns) == turns and new._args[1:] == rot._args[1:] == (64, 1, rot.magnitude)
    assert (new.head_dim, new.frequencies) == (128, rot.frequencies)


# ---------------------------------------------------------------- C ABI


def _rotate(**kw):
    a = dict(q=PTR, qs=256, k=PTR, ks=128, pos=None, turns=(ctypes.c_uint64 * 32)(*[1] * 32),
             dtype=1, tokens=3, seq=3, hq=4, hkv=2, d=64, r=64, inter=0, mu=1.0, back=0, qo=PTR,
             ko=PTR)
    a.update(kw)
    return L.mf_rotate(*a.values(), None)


@pytest.mark.parametrize("kw, code, text", [
    (dict(dtype=9), _lib.ERR_DTYPE, "dtype"),
    (dict(tokens=0), _lib.ERR_INVALID_ARGUMENT, "positive"),
    (dict(seq=0), _lib.ERR_INVALID_ARGUMENT, "positive"),
    (dict(hq=-1), _lib.ERR_INVALID_ARGUMENT, "positive"),
    (dict(d=63), _lib.ERR_HEAD_DIM, "head_dim"),
    (dict(d=2048), _lib.ERR_HEAD_DIM, "head_dim"),
    (dict(r=66), _lib.ERR_SHAPE, "rotary_dim"),
    (dict(r=7), _lib.ERR_SHAPE, "rotary_dim"),
    (dict(q=None), _lib.ERR_INVALID_ARGUMENT, "null"),
    (dict(hkv=0), _lib.ERR_INVALID_ARGUMENT, "null"),
    (dict(hkv=65535), _lib.ERR_SHAPE, "65535"),
    (dict(turns=None), _lib.ERR_INVALID_ARGUMENT, "turns"),
    (dict(mu=float("inf")), _lib.ERR_INVALID_ARGUMENT, "magnitude"),
    (dict(qs=255), _lib.ERR_SHAPE, "between tokens"),
    (dict(ks=-128), _lib.ERR_SHAPE, "between tokens"),
])
def test_rotate_abi_refuses(kw, code, text):
    assert _rotate(**kw) == code
    assert text in _msg()


def test_turns_of_frequencies():
    freqs = [1.0, 2 * math.pi, -1.0, 0.0, 1e-9, 2 * math.pi * 5.25, 1e6]
    turns = (ctypes.c_uint64 * 7)()
    assert L.mf_rotary_turns((ctypes.c_double * 7)(*freqs), 7, turns) == _lib.OK
    # 2^-64ths of a turn; a double holds f / 2 pi to 2^-53 of it, modulo whole turns
    for f, t in zip(freqs, turns):
        exact = f / (2 * math.pi) % 1.0
        off = abs(t / 2.0 ** 64 - exact)
        assert min(off, 1 - off) <= 2.0 ** -52 * max(1.0, abs(f)), (f, t)
    assert L.mf_rotary_turns((ctypes.c_double * 1)(float("nan")), 1, turns) == _lib.ERR_INVALID_ARGUMENT
    assert "finite" in _msg()
    assert L.mf_rotary_turns(None, 1, turns) == _lib.ERR_INVALID_ARGUMENT
    assert L.mf_rotary_turns((ctypes.c_double * 1)(1.0), 0, turns) == _lib.ERR_INVALID_ARGUMENT


def _strides(*s):
    return (ctypes.c_longlong * 3)(*s)


def _paged_plan(**kw):
    a = dict(starts=PTR, contexts=PTR, table=PTR, stride=8, r=2, n=4, width=8, ps=16, pages=9, hq=4,
             hkv=2, dtype=1, plan=PTR, nbytes=1 << 30)
    a.update(kw)
    return L.mf_paged_plan(*a.values(), None)


PAGED = [
    (dict(dtype=5), _lib.ERR_DTYPE, "dtype"),
    (dict(r=0), _lib.ERR_INVALID_ARGUMENT, "positive"),
    (dict(n=0), _lib.ERR_INVALID_ARGUMENT, "positive"),
    (dict(r=5000), _lib.ERR_SHAPE, "4096 sequences"),
    (dict(hq=3), _lib.ERR_HEADS, "divisible"),
    (dict(n=1 << 25, hq=4), _lib.ERR_SHAPE, "2^26"),
    (dict(hq=2048, hkv=2048), _lib.ERR_SHAPE, "1024"),
    (dict(ps=12), _lib.ERR_SHAPE, "multiple of 8"),
    (dict(ps=0), _lib.ERR_INVALID_ARGUMENT, "positive"),
    (dict(pages=0), _lib.ERR_INVALID_ARGUMENT, "positive"),
    (dict(plan=None), _lib.ERR_INVALID_ARGUMENT, "plan"),
    (dict(plan=ctypes.c_void_p((1 << 20) + 8)), _lib.ERR_INVALID_ARGUMENT, "aligned"),
    (dict(nbytes=64), _lib.ERR_WORKSPACE, "plan holds 64 bytes"),
]


@pytest.mark.parametrize("kw, code, text", PAGED + [
    (dict(width=0), _lib.ERR_SHAPE, "max_pages"),
    (dict(stride=7), _lib.ERR_SHAPE, "max_pages"),
    (dict(width=1 << 27, stride=1 << 27), _lib.ERR_SHAPE, "2^30"),
    (dict(r=4096, width=1 << 24, stride=1 << 24, ps=64), _lib.ERR_SHAPE, "too many for one step"),
    (dict(starts=None), _lib.ERR_INVALID_ARGUMENT, "non-null"),
    (dict(table=None), _lib.ERR_INVALID_ARGUMENT, "non-null"),
])
def test_plan_abi_refuses(kw, code, text):
    assert _paged_plan(**kw) == code
    assert text in _msg()


def _append(**kw):
    a = dict(q=PTR, qs=256, k=PTR, ks=128, v=PTR, vs=128, qg=PTR, kg=PTR, eps=1e-5,
             turns=(ctypes.c_uint64 * 32)(*[1] * 32), rd=64, inter=0, mu=1.0, dtype=1, n=4, r=2, hq=4,
             hkv=2, d=64, ps=16, pages=9, plan=PTR, nbytes=1 << 30, kp=PTR, vp=PTR,
             kst=_strides(2048, 128, 64), vst=_strides(2048, 128, 64), qo=PTR)
    a.update(kw)
    return L.mf_paged_append(*a.values(), None)


@pytest.mark.parametrize("kw, code, text", PAGED + [
    (dict(d=128), _lib.ERR_HEAD_DIM, "head_dim"),
    (dict(k=None), _lib.ERR_INVALID_ARGUMENT, "non-null"),
    (dict(q=None), _lib.ERR_INVALID_ARGUMENT, "both"),
    (dict(q=None, qo=None), _lib.ERR_INVALID_ARGUMENT, "both"),  # a gain without a query
    (dict(eps=-1.0), _lib.ERR_INVALID_ARGUMENT, "eps"),
    (dict(eps=float("nan")), _lib.ERR_INVALID_ARGUMENT, "eps"),
    (dict(rd=128), _lib.ERR_SHAPE, "rotary_dim"),
    (dict(vs=64), _lib.ERR_SHAPE, "between tokens"),
    (dict(kst=None), _lib.ERR_INVALID_ARGUMENT, "strides"),
    (dict(kst=_strides(2048, 32, 64)), _lib.ERR_SHAPE, "overlap"),
    (dict(vst=_strides(2048, 128, 0)), _lib.ERR_SHAPE, "overlap"),
    (dict(vst=_strides(-2048, 128, 64)), _lib.ERR_SHAPE, "overlap"),
    (dict(vst=_strides(2048, 1 << 27, 64)), _lib.ERR_SHAPE, "2^26"),
    (dict(kst=_strides(2048, 128, 1 << 30)), _lib.ERR_SHAPE, "2^29"),
    # pages that are written have slots of their own
    (dict(kst=_strides(0, 128, 64)), _lib.ERR_SHAPE, "overlap"),
    (dict(vst=_strides(1024, 128, 64)), _lib.ERR_SHAPE, "overlap"),
    (dict(vst=_strides(2048, 64, 64)), _lib.ERR_SHAPE, "overlap"),
    (dict(vst=_strides(2048, 64, 1000)), _lib.ERR_SHAPE, "overlap"),
    (dict(kst=_strides(64, 128, 64)), _lib.ERR_SHAPE, "overlap"),
    (dict(kst=_strides(1 << 62, 128, 64)), _lib.ERR_SHAPE, "between"),
])
def test_append_abi_refuses(kw, code, text):
    assert _append(**kw) == code
    assert text in _msg()


def _attn(**kw):
    a = dict(q=PTR, qs=256, kp=PTR, vp=PTR, kst=_strides(2048, 128, 64), vst=_strides(2048, 128, 64),
             table=PTR, stride=8, dtype=1, n=4, r=2, width=8, ps=16, pages=9, hq=4, hkv=2, d=64,
             scale=0.125, plan=PTR, nbytes=1 << 30, zero=1, out=PTR, ws=PTR, wsb=1 << 40)
    a.update(kw)
    return L.mf_paged_attn(*a.values(), None)


@pytest.mark.parametrize("kw, code, text", PAGED + [
    (dict(d=32), _lib.ERR_HEAD_DIM, "head_dim"),
    (dict(scale=0.0), _lib.ERR_INVALID_ARGUMENT, "scale"),
    (dict(scale=float("nan")), _lib.ERR_INVALID_ARGUMENT, "scale"),
    (dict(out=None), _lib.ERR_INVALID_ARGUMENT, "non-null"),
    (dict(ws=None), _lib.ERR_INVALID_ARGUMENT, "non-null"),
    (dict(width=0), _lib.ERR_SHAPE, "max_pages"),
    (dict(kst=_strides(2048, 132, 64)), _lib.ERR_SHAPE, "16-byte"),
    (dict(qs=260), _lib.ERR_SHAPE, "16-byte"),
    (dict(kp=ctypes.c_void_p((1 << 20) + 8)), _lib.ERR_SHAPE, "16-byte"),
    (dict(wsb=16), _lib.ERR_WORKSPACE, "workspace holds 16"),
])
def test_attention_abi_refuses(kw, code, text):
    assert _attn(**kw) == code
    assert text in _msg()


def test_sizes_of_plan_and_workspace():
    # more tokens, sequences or heads never need less
    last = 0
    for n in (1, 2, 64, 1000, 40000):
        p = L.mf_paged_plan_bytes(64, n, 16, 8, 1)
        w = L.mf_paged_attn_workspace_bytes(64, n, 16, 8, 1)
        assert p > 0 and w > 0 and p + w > last
        last = p + w
    for sizes in ((0, 1, 16, 8), (5000, 1, 16, 8), (1, 1, 16, 3), (1, 1, 2, 4), (1, 1 << 23, 16, 8),
                  (1, 1, 2048, 2048), (2, 0, 16, 8), (-1, 4, 16, 8)):
        assert L.mf_paged_plan_bytes(*sizes, 1) == L.mf_paged_attn_workspace_bytes(*sizes, 0) == 0
    assert L.mf_paged_plan_bytes(0, 1, 16, 8, 1) == 0
    assert L.mf_paged_attn_workspace_bytes(1, 1, 0, 8, 1) == 0
