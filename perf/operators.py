"""Serving operators over a paged key/value cache, and the rotary embedding, as cases.

A case is one pass through an operator: ``rotate`` (rotary embedding of queries
and keys, with its backward pass in training), ``append`` (new keys and values
into the pages, per-head norm and rotation on the way), ``attend`` (attention of
every sequence's new tokens over its pages) or ``step`` (append, then attend, as
one layer of a serving step makes them).  Sizes are those of the framework's own
layouts (16 query and 8 key heads of 64, rows of 4096 packed tokens, 64 caches of
up to 8192 slots) with the smaller, longer and odd ones around them.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges,
``prepare`` makes what a program holds before the call, ``run`` is the call: in
elementary operations where ``own`` is false, through the framework where it is
true.  ``exact`` is the operators' definition in 64 bits.
"""

from __future__ import annotations

import math
import pathlib
import sys

import numpy as np
import torch

own = False

D = 64  # head dimension of the cached attention
_DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
_BYTES = {"bfloat16": 2, "float32": 4}
_EPS = 1e-5


# --------------------------------------------------------------------------- cases


def _turn(dim, part, interleaved, theta, scaling, factor, original):
    """A rotary embedding: ``part`` of a head's ``dim`` dims rotate."""
    return {"dim": dim, "part": part, "interleaved": interleaved, "theta": theta,
            "scaling": scaling, "factor": factor, "original": original}


def _rotate(dtype, rows, tokens, heads, kv_heads, offset, train, turn):
    return {"kind": "rotate", "dtype": dtype, "rows": rows, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "offset": offset, "train": train, **turn}


def _cached(kind, dtype, singles, chunks, new, before, heads, kv_heads, page, head_major, layout,
            norm=True, turn=None):
    """``singles`` sequences with one new token and ``chunks`` with ``new`` (low, high), each
    behind ``before`` (low, high) cached tokens, in pages of ``page`` tokens.  ``head_major``:
    a page holds one head's tokens next to each other, not one token's heads."""
    return {"kind": kind, "dtype": dtype, "singles": singles, "chunks": chunks, "new_low": new[0],
            "new_high": new[1], "before_low": before[0], "before_high": before[1], "heads": heads,
            "kv_heads": kv_heads, "page": page, "head_major": head_major, "layout": layout,
            "norm": norm, **(turn or _turn(D, D, False, 1e6, "none", 1.0, 0))}


def listed():
    return [
        # rotary embedding of a packed training step at the framework's headline
        # layout, forward and backward, frequencies stretched for a longer context
        {"name": "rotate_train",
         **_rotate("bfloat16", 8, 4096, 16, 8, 0, True,
                   _turn(64, 64, False, 1e6, "bands", 8.0, 8192))},
        # a float32 check of a model that rotates neighbours in a quarter of a wider
        # head, short odd rows
        {"name": "rotate_fp32_part",
         **_rotate("float32", 3, 333, 12, 4, 1000, True,
                   _turn(128, 32, True, 1e4, "none", 1.0, 0))},
        # the new tokens of a decode step of a serving batch: launches
        {"name": "append_step",
         **_cached("append", "bfloat16", 64, 0, (1, 1), (127, 8191), 16, 8, 16, False, 404)},
        # the tokens of several prompts at once: bandwidth
        {"name": "append_prompts",
         **_cached("append", "bfloat16", 0, 6, (512, 6000), (0, 2000), 16, 8, 64, False, 21)},
        # float32, no norm, half of the head rotated as neighbours far into a long
        # context, an odd page size
        {"name": "append_fp32",
         **_cached("append", "float32", 3, 4, (1, 301), (90000, 131000), 12, 4, 24, True, 22, False,
                   _turn(64, 32, True, 1e4, "linear", 4.0, 0))},
        # one user's next token: latency
        {"name": "attend_one",
         **_cached("attend", "bfloat16", 1, 0, (1, 1), (2000, 4095), 16, 8, 16, False, 15)},
        # a serving batch's next tokens over ragged contexts: bandwidth
        {"name": "attend_batch",
         **_cached("attend", "bfloat16", 64, 0, (1, 1), (127, 8191), 16, 8, 16, False, 404)},
        # two users with book-long contexts: few rows, the keys must be split
        {"name": "attend_long",
         **_cached("attend", "bfloat16", 2, 0, (1, 1), (120000, 131071), 32, 8, 64, True, 16)},
        # drafted tokens checked against the cache, a few per sequence
        {"name": "attend_drafts",
         **_cached("attend", "bfloat16", 0, 24, (3, 8), (1000, 16000), 24, 8, 32, False, 17)},
        # a chunk of a long prompt behind what is cached of it: matrix products
        {"name": "attend_chunk",
         **_cached("attend", "bfloat16", 0, 1, (2048, 2048), (28672, 28672), 16, 8, 64, False, 18)},
        # a float32 reference for a bf16 server: ragged chunks and single tokens
        {"name": "attend_fp32",
         **_cached("attend", "float32", 5, 3, (0, 200), (0, 1500), 8, 2, 24, False, 19)},
        # one layer of a continuously batched step: decoding users and arriving
        # prompts together, append and attention
        {"name": "step_mixed",
         **_cached("step", "bfloat16", 40, 3, (300, 1400), (100, 7000), 16, 8, 16, False, 20)},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


_HEADS = ((16, 8), (16, 8), (32, 8), (8, 8), (24, 8), (12, 4), (8, 1))
_PAGES = (16, 16, 32, 64, 128, 24, 40)


def _draw_turn(rng, dim):
    part = rng.choice((dim, dim, dim // 2, dim // 4))
    scaling = rng.choice(("none", "none", "linear", "base", "bands", "ramp"))
    factor = 1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0, 32.0))
    return _turn(dim, part, rng.random() < 0.4, rng.choice((1e4, 5e5, 1e6)), scaling, factor,
                 rng.choice((4096, 8192)) if scaling in ("bands", "ramp") else 0)


def draw(rng):
    """One more case: the listed kinds at sizes spread over their ranges."""
    kind = rng.choice(("rotate", "append", "attend", "attend", "attend", "step"))
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    heads, kv_heads = rng.choice(_HEADS)
    if kind == "rotate":
        turn = _draw_turn(rng, rng.choice((64, 64, 128, 96)))
        tokens = _log_int(rng, 16, 4096)
        most = 32768 * 24 * 128 // ((heads + kv_heads) * turn["dim"] * _BYTES[dtype])
        rows = max(1, _log_int(rng, 16, most) // tokens)
        return _rotate(dtype, rows, tokens, heads, kv_heads, rng.choice((0, 0, 5000, 120000)),
                       rng.random() < 0.7, turn)
    while True:
        singles = rng.choice((0, 0, 1, _log_int(rng, 1, 64)))
        chunks = 0 if singles and rng.random() < 0.4 else _log_int(rng, 1, 24)
        high = _log_int(rng, 1, 4096)
        low = rng.choice((0, 1, max(1, high // 4)))
        before = _log_int(rng, 1, 131071)
        case = _cached(kind, dtype, singles, chunks, (low, high),
                       (rng.choice((0, before // 8, before)), before), heads, kv_heads,
                       rng.choice(_PAGES), rng.random() < 0.4, rng.randrange(1 << 30),
                       rng.random() < 0.7, _draw_turn(rng, D))
        spans, w = _spans(case), work(case)
        # no more than the largest listed cases cost, nor a pool of more than 0.9 GB
        grid = sum(int(n) * int(c) for n, c in spans) * heads
        if (spans[:, 0].sum() and w["flops"] <= (4e10 if dtype == "float32" else 2.6e11)
                and spans[:, 0].sum() <= 24000 and w["bytes"] <= 5.5e8 and grid <= 2e9
                and spans[:, 1].max() * len(spans) * kv_heads * _BYTES[dtype] <= 2e7):
            return case


# --------------------------------------------------------------------------- layouts


def _spans(case):
    """[sequences, 2]: new tokens and context length (new tokens included) of each sequence."""
    rng = np.random.default_rng(case["layout"])
    new = np.concatenate((np.ones(case["singles"], np.int64),
                          rng.integers(case["new_low"], case["new_high"] + 1, size=case["chunks"])))
    before = rng.integers(case["before_low"], case["before_high"] + 1, size=len(new))
    return np.stack((new, before + new), 1)[rng.permutation(len(new))]


def _frequencies(case):
    """Radians per position of every rotated pair, in 64 bits, and the factor of the result."""
    r, s = case["part"], case["factor"]
    i = torch.arange(0, r // 2, dtype=torch.float64)
    theta = case["theta"] * s ** (r / (r - 2)) if case["scaling"] == "base" else case["theta"]
    f, magnitude = theta ** (-2 * i / r), 1.0
    if case["scaling"] == "linear":
        f = f / s
    elif case["scaling"] == "bands":
        # by turns in the original length: above 4 kept, below 1 slowed, between blended
        turns = case["original"] * f / (2 * math.pi)
        keep = ((turns - 1) / 3).clamp(0, 1)
        f = f * (keep + (1 - keep) / s)
    elif case["scaling"] == "ramp":
        # by index: from the pair with 32 turns in the original length to that with one
        lo, hi = (r * math.log(case["original"] / (2 * math.pi * n)) / (2 * math.log(theta))
                  for n in (32, 1))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), r - 1)
        slow = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f * (1 - slow + slow / s)
        magnitude = 1 + 0.1 * math.log(s)
    return f, magnitude


# --------------------------------------------------------------------------- inputs


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    h, kvh = case["heads"], case["kv_heads"]
    state = {"case": case}

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev, dtype=dtype)

    f, state["magnitude"] = _frequencies(case)
    state["frequencies"] = f.to(dev)
    if case["kind"] == "rotate":
        b, t, d = case["rows"], case["tokens"], case["dim"]
        # queries and keys are parts of one projection, as a layer's fused product leaves them
        fused = normal(b, t, (h + 2 * kvh) * d)
        state["q"] = fused[..., :h * d].unflatten(-1, (h, d))
        state["k"] = fused[..., h * d:(h + kvh) * d].unflatten(-1, (kvh, d))
        # every row starts at a place of its own in its document
        first = torch.randint(0, 1 + case["offset"], (b, 1), generator=gen, device=dev)
        state["positions"] = (first + torch.arange(t, device=dev)).to(torch.int32)
        if case["train"]:
            state["dq"], state["dk"] = normal(b, t, h, d), normal(b, t, kvh, d)
            for name in ("q", "k"):
                state[name].requires_grad_()
        return state
    spans, ps = _spans(case), case["page"]
    per = -(-spans[:, 1] // ps)  # pages of each sequence
    used, widest = int(per.sum()), max(1, int(per.max()))
    # the pool's pages come in any order, some are nobody's
    pages = used + max(2, used // 20)
    order = np.random.default_rng([case["layout"], seed]).permutation(pages)
    table = np.full((len(spans), widest), -1, np.int32)
    table[np.arange(widest)[None] < per[:, None]] = order[:used]
    state["page_table"] = torch.from_numpy(table).to(dev)
    state["query_starts"] = torch.from_numpy(np.concatenate(([0], np.cumsum(spans[:, 0]))).astype(np.int32)).to(dev)
    state["context_lengths"] = torch.from_numpy(spans[:, 1].astype(np.int32)).to(dev)
    n = int(spans[:, 0].sum())
    if case["head_major"]:
        pool = normal(2, pages, kvh, ps, D).transpose(2, 3)
    else:
        pool = normal(2, pages, ps, kvh, D)
    state["key_pages"], state["value_pages"] = pool[0], pool[1]
    if case["kind"] == "attend":
        state["q"] = normal(n, h, D)  # unit-variance heads, as the norm leaves them
        return state
    fused = normal(n, (h + 2 * kvh) * D)
    state["q"] = fused[:, :h * D].unflatten(-1, (h, D))
    state["k"] = fused[:, h * D:(h + kvh) * D].unflatten(-1, (kvh, D))
    state["v"] = fused[:, (h + kvh) * D:].unflatten(-1, (kvh, D))
    if case["norm"]:
        for name in ("q_gain", "k_gain"):
            state[name] = (1 + 0.1 * torch.randn(D, generator=gen, device=dev)).to(dtype)
    return state


# --------------------------------------------------------------------------- the call


def run(state):
    case = state["case"]
    if own:
        return _call(case, state)
    if case["kind"] == "rotate":
        return _plain_rotate(case, state)
    res = {}
    if case["kind"] != "attend":
        q = _plain_append(case, state)
        res = {"key_pages": state["key_pages"], "value_pages": state["value_pages"]}
        if case["kind"] == "append":
            return {"q": q, **res}
    else:
        q = state["q"]
    return {"out": _plain_attend(case, state, q), **res}


def _call(case, s):
    """The same pass through the framework."""
    package = str(pathlib.Path(__file__).resolve().parents[1] / "minifield-training_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from mfattn.kernels import paged, rotary

    turn = s.get("rotary")
    if turn is None:  # a model's own, made once from its configuration
        turn = s["rotary"] = rotary.Rotary(
            case["dim"], theta=case["theta"], rotary_dim=case["part"],
            interleaved=case["interleaved"], scaling=case["scaling"], factor=case["factor"],
            original_length=case["original"] or None)
    if case["kind"] == "rotate":
        q, k = rotary.rotate(s["q"], s["k"], turn, s["positions"])
        if not case["train"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    # every step brings its own lengths and pages: its plan is part of the pass
    plan = paged.plan(s["query_starts"], s["context_lengths"], s["page_table"], s["key_pages"],
                      tokens=s["q"].shape[0], query_heads=case["heads"])
    res, q = {}, s["q"]
    if case["kind"] != "attend":
        q = paged.append(s["k"], s["v"], s["key_pages"], s["value_pages"], plan, query=q,
                         rotary=turn, query_gain=s.get("q_gain"), key_gain=s.get("k_gain"),
                         eps=_EPS)
        res = {"key_pages": s["key_pages"], "value_pages": s["value_pages"]}
        if case["kind"] == "append":
            return {"q": q, **res}
    return {"out": paged.attention(q, s["key_pages"], s["value_pages"], plan), **res}


# --------------------------------------------------------------------------- plain forms


def _rotated(x, cos, sin, case):
    """The first ``part`` dims of x (float32) turned by the angles, pairs by the case's layout."""
    r = case["part"]
    turned, rest = x[..., :r], x[..., r:]
    if case["interleaved"]:
        u, w = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack((u * cos - w * sin, w * cos + u * sin), -1).flatten(-2)
    else:
        u, w = turned[..., :r // 2], turned[..., r // 2:]
        y = torch.cat((u * cos - w * sin, w * cos + u * sin), -1)
    return torch.cat((y, rest), -1)


def _cos_sin(s, positions):
    # far positions have angles of many turns: 64 bits
    a = positions.double()[..., None, None] * s["frequencies"]
    return ((f(a) * s["magnitude"]).float() for f in (torch.cos, torch.sin))


def _plain_rotate(case, s):
    dtype = s["q"].dtype
    cos, sin = _cos_sin(s, s["positions"])
    res = {n: _rotated(s[n].detach().float(), cos, sin, case).to(dtype) for n in ("q", "k")}
    if case["train"]:
        # the rotation's transpose turns back
        res.update((n, _rotated(s[n].float(), cos, -sin, case).to(dtype)) for n in ("dq", "dk"))
    return res


def _plain_tokens(s):
    """Sequence and position of every new token."""
    starts = s["query_starts"].long()
    token = torch.arange(s["q"].shape[0], device=starts.device)
    seq = torch.searchsorted(starts[1:], token, right=True)
    return seq, s["context_lengths"].long()[seq] - starts[seq + 1] + token


def _plain_append(case, s):
    dtype = s["q"].dtype
    seq, position = _plain_tokens(s)
    cos, sin = _cos_sin(s, position)

    def turned(x, gain):
        x = x.float()
        if gain is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * gain.float()
        return _rotated(x, cos, sin, case).to(dtype)

    page, slot = s["page_table"].long()[seq, position // case["page"]], position % case["page"]
    s["key_pages"][page, slot] = turned(s["k"], s.get("k_gain"))
    s["value_pages"][page, slot] = s["v"]
    return turned(s["q"], s.get("q_gain"))


def _plain_attend(case, s, q):
    spans = _spans(case)
    out = torch.zeros_like(q)
    for group in (spans[:, 0] == 1, spans[:, 0] > 1):  # one token each; padded to the longest
        which = np.flatnonzero(group)
        if len(which):
            _plain_attend_group(case, s, q, out, torch.from_numpy(which).to(q.device),
                                int(spans[which, 0].max()), int(spans[which, 1].max()))
    return out


def _plain_attend_group(case, s, q, out, which, most, longest):
    group, kvh, dev = case["heads"] // case["kv_heads"], case["kv_heads"], q.device
    starts, context = s["query_starts"].long(), s["context_lengths"].long()[which]
    first, count = starts[which], starts[which + 1] - starts[which]
    i, j = torch.arange(most, device=dev), torch.arange(longest, device=dev)
    page = s["page_table"].long()[which][:, j // case["page"]].clamp(min=0)
    k = s["key_pages"][page, j % case["page"]].float()    # [sequences, keys, heads, D]
    v = s["value_pages"][page, j % case["page"]].float()
    gone = j[None] >= context[:, None]  # slots behind a context hold anything
    v = v.masked_fill(gone[..., None, None], 0)
    real = i[None] < count[:, None]
    token = (first[:, None] + i[None]).clamp(max=q.shape[0] - 1)
    x = q[token].float().unflatten(2, (kvh, group))
    x = x.permute(0, 2, 3, 1, 4).flatten(2, 3)             # [sequences, heads, group * new, D]
    scores = torch.matmul(x, k.permute(0, 2, 3, 1).contiguous()) * D ** -0.5
    seen = j[None, None] <= (context - count)[:, None, None] + i[None, :, None]
    seen &= ~gone[:, None]
    scores = scores.unflatten(2, (group, most)).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top.masked_fill(top == -math.inf, 0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v.transpose(1, 2).contiguous()).unflatten(2, (group, most))
    o = o / total.masked_fill(total == 0, 1)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)             # [sequences, new, heads, D]
    out[token[real]] = o[real].to(q.dtype)


# --------------------------------------------------------------------------- work


def work(case):
    size, h, kvh = _BYTES[case["dtype"]], case["heads"], case["kv_heads"]
    if case["kind"] == "rotate":
        tokens = case["rows"] * case["tokens"]
        values = tokens * (h + kvh) * case["dim"] * (2 if case["train"] else 1)
        return {"bytes": 2 * values * size + 4 * tokens, "flops": 3 * values}
    spans, ps = _spans(case), case["page"]
    n, context = int(spans[:, 0].sum()), int(spans[spans[:, 0] > 0, 1].sum())
    plan = 4 * (2 * len(spans) + 1)
    # queries in, queries or outputs out; new keys and values in and into their pages
    nbytes, flops = 2 * n * h * D * size + plan, 0
    if case["kind"] != "attend":
        nbytes += 4 * n * kvh * D * size + 4 * n
        flops += n * (h + kvh) * D * (8 if case["norm"] else 3)
    if case["kind"] != "append":
        nbytes += 2 * context * kvh * D * size + 4 * int((-(-spans[:, 1] // ps)).sum())
        pairs = sum(int(m) * (int(c) - int(m)) + int(m) * (int(m) + 1) // 2 for m, c in spans)
        flops += 4 * D * h * pairs
    return {"bytes": nbytes, "flops": flops}


# --------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "rotate":
            return _exact_rotate(case, s)
        keys, values = s["key_pages"].double(), s["value_pages"].double()
        spans, starts = _spans(case).tolist(), s["query_starts"].tolist()
        table, q = s["page_table"].long(), s["q"].double()
        res = {}
        if case["kind"] != "attend":
            q = _exact_append(case, s, spans, starts, table, keys, values)
            res = {"key_pages": keys, "value_pages": values}
            if case["kind"] == "append":
                return {"q": q, **res}
            # the attention reads what the append rounded
            dtype = s["q"].dtype
            q, keys, values = (x.to(dtype).double() for x in (q, keys, values))
        return {"out": _exact_attend(case, spans, starts, table, q, keys, values), **res}


def _exact_turn(case, s, x, positions, back=False):
    """Pairs as complex numbers times magnitude * e^(i angle)."""
    r = case["part"]
    angle = positions.double()[..., None] * s["frequencies"]
    unit = torch.polar(torch.full_like(angle, s["magnitude"]), -angle if back else angle)
    shape = (r // 2, 2) if case["interleaved"] else (2, r // 2)
    pair = x[..., :r].unflatten(-1, shape)
    if not case["interleaved"]:
        pair = pair.transpose(-1, -2)
    y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * unit[..., None, :])
    if not case["interleaved"]:
        y = y.transpose(-1, -2)
    y = y.flatten(-2)
    return torch.cat((y, x[..., r:]), -1)


def _exact_rotate(case, s):
    res = {n: _exact_turn(case, s, s[n].detach().double(), s["positions"]) for n in ("q", "k")}
    if case["train"]:
        for n in ("dq", "dk"):
            res[n] = _exact_turn(case, s, s[n].double(), s["positions"], back=True)
    return res


def _exact_append(case, s, spans, starts, table, keys, values):
    q = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for r, (n, context) in enumerate(spans):
        at = slice(starts[r], starts[r] + n)
        position = torch.arange(context - n, context, device=q.device)
        page, slot = table[r, position // case["page"]], position % case["page"]
        q[at], keys[page, slot] = (
            _exact_turn(case, s, x if g is None else
                        x / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS) * g.double(), position)
            for x, g in ((s["q"][at].double(), s.get("q_gain")), (s["k"][at].double(), s.get("k_gain"))))
        values[page, slot] = s["v"][at].double()
    return q


def _exact_attend(case, spans, starts, table, q, keys, values):
    out, group = torch.zeros_like(q), case["heads"] // case["kv_heads"]
    for r, (n, context) in enumerate(spans):
        if n == 0:
            continue
        at = slice(starts[r], starts[r] + n)
        j = torch.arange(context, device=q.device)
        k, v = (x[table[r, j // case["page"]], j % case["page"]].transpose(0, 1) for x in (keys, values))
        hidden = j[None] > torch.arange(context - n, context, device=q.device)[:, None]
        for head in range(case["heads"]):
            w = torch.matmul(q[at, head], k[head // group].t()) * D ** -0.5
            w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
            out[at, head] = torch.matmul(w, v[head // group])
    return out
