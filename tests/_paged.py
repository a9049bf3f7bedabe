"""Paged batches of the serving tests, and their definition in 64 bits.

``Batch`` lays ragged sequences out over a shuffled page pool; ``attend`` and
``turned`` are the attention and the (norm and) rotation in float64, written
from the formulas, one sequence and head at a time, with the magnitudes that
the tests' error bounds are made of.
"""

from __future__ import annotations

import math

import numpy as np
import torch

EPS24 = 2.0 ** -24  # half a step of float32, relative
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


class Batch:
    """``spans``: (new tokens, context) of each sequence."""

    def __init__(self, spans, hq, hkv, page_size, dtype, device, *, seed=0, layout="slots",
                 spare=3, behind=0, width=0, spread=3.0):
        rng = np.random.default_rng(seed)
        gen = torch.Generator(device=device).manual_seed(seed)
        self.spans, self.hq, self.hkv, self.ps, self.dtype = spans, hq, hkv, page_size, dtype
        self.device = device
        per = [-(-c // page_size) for _, c in spans]
        self.width = max(1, width, *per)
        pages = sum(per) + spare
        order = rng.permutation(pages).astype(np.int32)
        table = np.full((len(spans), self.width), -1, np.int32)
        at = 0
        for r, n in enumerate(per):
            table[r, :n] = order[at:at + n]
            at += n
        self.table = table
        self.starts = np.concatenate(([0], np.cumsum([n for n, _ in spans]))).astype(np.int32)
        self.tokens = int(self.starts[-1]) + behind
        self.contexts = np.array([c for _, c in spans], np.int32)

        def normal(*shape, scale=1.0):
            return (torch.randn(shape, generator=gen, device=device) * scale).to(dtype)

        if layout == "slots":       # [page][slot][head]
            pool = normal(2, pages, page_size, hkv, 64)
        elif layout == "heads":     # [page][head][slot]
            pool = normal(2, pages, hkv, page_size, 64).transpose(2, 3)
        elif layout == "together":  # keys and values of a slot side by side
            pool = normal(pages, page_size, 2, hkv, 64).permute(2, 0, 1, 3, 4)
        elif layout == "apart":     # keys by slots, values by heads
            pool = (normal(pages, page_size, hkv, 64),
                    normal(pages, hkv, page_size, 64).transpose(1, 2))
        else:
            raise KeyError(layout)
        self.key_pages, self.value_pages = pool[0], pool[1]
        # scores of standard deviation `spread`: the softmax rests on few keys, so
        # a key too many or too few shows
        self.q = normal(self.tokens, hq, 64, scale=spread)
        self.k, self.v = normal(self.tokens, hkv, 64), normal(self.tokens, hkv, 64)

    def on_device(self):
        return tuple(torch.from_numpy(x).to(self.device)
                     for x in (self.starts, self.contexts, self.table))

    def plan(self):
        from mfattn.kernels import paged

        starts, contexts, table = self.on_device()
        return paged.plan(starts, contexts, table, self.key_pages, tokens=self.tokens,
                          query_heads=self.hq)

    def slots(self, r, positions):
        """Pages (-1: none) and slots of positions of sequence r."""
        page = self.table[r][np.asarray(positions) // self.ps].astype(np.int64)
        page[(page < 0) | (page >= self.key_pages.shape[0])] = -1
        return page, np.asarray(positions) % self.ps


def attend(batch: Batch, q, key_pages, value_pages, scale=0.125):
    """(out, bound): the definition in float64 and the error that a result may have.

    With S = sum |q k| scale over a row's dims, a score is off by at most 65
    half steps of float32 of S (64 products and sums, the scale), a weight by
    twice that relative to the others, plus 8 half steps for the exponential and
    the shift; sums of n weights add n half steps.  In bf16 the weights are
    rounded once, above and below the fraction alike (2 * 2^-8 together), and the
    result is rounded once.
    """
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros_like(out)
    group = batch.hq // batch.hkv
    q64 = q.double().cpu()
    pool_k, pool_v = key_pages.cpu(), value_pages.cpu()
    for r, (n, context) in enumerate(batch.spans):
        if n == 0:
            continue
        reach = min(context, batch.width * batch.ps)
        pos = np.arange(reach)
        page, slot = batch.slots(r, pos) if reach else (np.zeros(0, np.int64),) * 2
        there = torch.from_numpy(page >= 0)
        k = pool_k[np.maximum(page, 0), slot].double()
        v = pool_v[np.maximum(page, 0), slot].double()
        at = torch.arange(int(batch.starts[r]), int(batch.starts[r]) + n)
        sees = torch.from_numpy(pos)[None] <= (torch.arange(n) + context - n)[:, None]
        sees = sees & there[None]
        for h in range(batch.hq):
            kh, vh = k[:, h // group], v[:, h // group]
            qh = q64[at, h]
            for i in range(n):
                w = sees[i]
                if not bool(w.any()):
                    continue
                s = (kh[w] @ qh[i]) * scale
                mag = ((kh[w].abs() @ qh[i].abs()) * scale).max().item()
                p = torch.softmax(s, 0)
                o, big = p @ vh[w], p @ vh[w].abs()
                out[at[i], h] = o
                rel = (2 * 65 * mag + 8 + int(w.sum())) * EPS24
                if batch.dtype is torch.bfloat16:
                    rel += 2 * HALF_STEP[torch.bfloat16]
                bound[at[i], h] = rel * big + HALF_STEP[batch.dtype] * o.abs()
    return out, bound


def turned(x, positions, rotary, gain=None, eps=1e-5, back=False, dtype=None):
    """(y, bound) of rotated (and, with a gain, normalised) heads in float64.

    In half steps of float32, relative to magnitude * (|u| + |w|) of a pair: the
    angle's conversion pi / 2 and its truncation, cos and sin 4, the magnitude
    1, the products 1, their sum 1: at most 10.  The norm before it: the sum of
    64 squares at most 64 / 4 + 4 in a chain and a tree, halved by the root, the
    root 2, two products: at most 16.  One rounding to the dtype on top.
    """
    dtype = x.dtype if dtype is None else dtype
    x = x.double().cpu()
    steps = 0
    if gain is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain.double().cpu()
        steps += 16
    y, mag = x.clone(), x.abs()
    if rotary is not None:
        half, mu = rotary.rotary_dim // 2, rotary.magnitude
        pos = torch.as_tensor(positions).cpu()
        for i, f in enumerate(rotary.frequencies):
            a, b = (2 * i, 2 * i + 1) if rotary.interleaved else (i, i + half)
            angle = pos.double() * f
            c, s = torch.cos(angle)[..., None] * mu, torch.sin(angle)[..., None] * mu
            s = -s if back else s
            u, w = x[..., a], x[..., b]
            y[..., a], y[..., b] = u * c - w * s, w * c + u * s
            mag[..., a] = mag[..., b] = mu * (u.abs() + w.abs())
        steps += 10
    return y, steps * EPS24 * mag + HALF_STEP[dtype] * y.abs()


def close(got, want, bound, what=""):
    """Every element within its bound (which counts roundings; nothing on top)."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    over = ((got - want).abs() - bound)
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0, f"{what}: {worst:.3e} beyond its bound"
    assert math.isfinite(worst)
