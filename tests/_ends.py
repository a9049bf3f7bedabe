"""Definitions in float64 of the norms, the embedding's gradient and the distillation
loss, with bounds on what float32 arithmetic may be off.

``E`` is half a step of float32.  A sum that adds at most ``depth`` terms in a row (a
lane's own, then the lanes', the waves' and the workgroups') is off by at most
``depth * E`` of the sum of the terms' sizes, to first order.
"""

from __future__ import annotations

import math

import torch

E = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
# a lane adds up to 64 of a row's values, then 6 sums over lanes and 8 waves
DEPTH = 64 + 6 + 8


def check(got, want, bound, what):
    """|got - want| within ``bound`` and half a step of the result's own dtype."""
    want = want.to(got.device)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    room = bound.to(got.device) + HALF_STEP[got.dtype] * (want.abs() + bound.to(got.device)) + 1e-37
    bad = ~(off <= room) & (got.double() != want)  # (infinities are equal, their difference is not 0)
    assert not bad.any(), (what, int(bad.sum()), float((off / room).nan_to_num(9e9).max()))


def norm(x, w, b, eps, center, dy=None):
    """{name: (value, bound)} of y and, with dy, of dx, dweight and dbias."""
    x, w = x.double(), w.double()
    d, rows = x.shape[-1], x.shape[0]
    mean = x.mean(-1, keepdim=True) if center else torch.zeros_like(x[:, :1])
    off = x - mean
    var = (off * off).mean(-1, keepdim=True)
    rstd = (var + eps) ** -0.5
    h = off * rstd
    # the mean: its sum, 1 / D and the product; a difference to it: its own rounding too
    mean_e = (DEPTH + 2) * E * x.abs().mean(-1, keepdim=True) if center else 0 * mean
    off_e = mean_e + E * off.abs()
    # the mean square: each square moves by 2 |off| off_e, its sum and 1 / D
    var_e = (2 * off.abs() * off_e + off_e ** 2).mean(-1, keepdim=True) + (DEPTH + 3) * E * var
    # -1/2 of the relative error, and two steps of the root; generous where the error is large
    rel = 0.5 * var_e / (var + eps) * (1 + var_e / (var + eps)) + 4 * E
    h_e = rstd * off_e * (1 + rel) + h.abs() * (rel + E)
    y = h * w + (b.double() if b is not None else 0)
    y_e = h_e * w.abs() + 3 * E * (h * w).abs() + E * y.abs()
    res = {"y": (y, y_e)}
    if dy is None:
        return res
    dy = dy.double()
    g = dy * w
    gm, gh = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    if not center:
        gm = 0 * gm
    gm_e = (DEPTH + 3) * E * g.abs().mean(-1, keepdim=True)
    gh_e = (g.abs() * h_e).mean(-1, keepdim=True) + (DEPTH + 4) * E * (g * h).abs().mean(-1, keepdim=True)
    inner = g - gm - h * gh
    inner_e = gm_e + h.abs() * gh_e + h_e * (gh.abs() + gh_e) + 4 * E * (
        g.abs() + gm.abs() + (h * gh).abs())
    res["dx"] = (rstd * inner, rstd * (inner_e * (1 + rel) + inner.abs() * (rel + 2 * E)))
    # the rows' sums: each term's own error, at most `rows` terms in a row, then 512 pieces
    deep = rows + 8 + 512
    res["dweight"] = ((dy * h).sum(0), (dy.abs() * h_e).sum(0) + deep * E * (dy * h).abs().sum(0))
    res["dbias"] = (dy.sum(0), deep * E * dy.abs().sum(0))
    return res


def embed_gradient(ids, dout, vocabulary, scale, padding=-1):
    """(value, bound) of the table's gradient."""
    d = dout.shape[-1]
    ids, dout = ids.reshape(-1).cpu(), dout.reshape(-1, d).double().cpu()
    real = (ids >= 0) & (ids < vocabulary) & (ids != padding)
    ids, dout = ids[real].long(), dout[real]
    grad = torch.zeros(vocabulary, d, dtype=torch.float64).index_add_(0, ids, dout) * scale
    size = torch.zeros(vocabulary, d, dtype=torch.float64).index_add_(0, ids, dout.abs()) * abs(scale)
    count = torch.zeros(vocabulary, dtype=torch.float64).index_add_(0, ids, torch.ones(len(ids)).double())
    return grad, (count[:, None] + 2) * E * size


def distill(z, teacher, ids, temperature=1.0, total=None, weights=None, upstream=None):
    """(loss, bound, gradient, bound) row by row."""
    rows, v = z.shape
    z, t = z.double().cpu(), teacher.double().cpu() / temperature
    ids = ids.cpu().long()
    loss, loss_e = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    grad, grad_e = torch.zeros_like(z), torch.zeros_like(z)
    for n in range(rows):
        w = 1.0 if weights is None else float(weights[n])
        here = (ids[n] >= 0) & (ids[n] < v)
        if w == 0 or (total is None and not (here & (t[n] > -torch.inf)).any()):
            continue
        at, u = ids[n][here], t[n][here]
        logp = u - (float(total[n]) if total is not None else torch.logsumexp(u, 0))
        p = logp.exp()
        rest = max(0.0, 1 - float(p.sum())) if total is not None else 0.0
        logq = torch.log_softmax(z[n] / temperature, 0)
        q = logq.exp()
        beyond = torch.ones(v, dtype=torch.bool)
        beyond[at] = False
        s = float(q[beyond].sum())
        kl = float(torch.where(p > 0, p * (logp - logq[at]), 0.0).sum())
        if rest > 0:
            kl += rest * (math.log(rest) - (math.log(s) if s > 0 else -math.inf))
        loss[n] = w * temperature ** 2 * kl
        # an exponential's argument z' = (z - max) / T has three roundings and the exponential
        # two steps; under q, |z'| is log V at most on average; a thread (one of 256 at least, of
        # 512 where the row is longer than 2^15) adds its share of the row, then 6 + 16 sums
        arg = (z[n] - z[n].max()).abs() / temperature
        arg = torch.where(q > 0, arg, 0.0)
        mean_arg = float((q * arg).sum())
        share = v // (256 if v <= 1 << 15 else 512)
        sums = (share + 8 + 22 + 4 + 3 * mean_arg) * E
        rest_arg = float((q * arg)[beyond].sum()) / s if s > 0 else 0.0
        rest_sums = (share + 8 + 22 + 4 + 3 * rest_arg) * E
        mass = float(p.sum()) + rest
        loss_e[n] = abs(w) * temperature ** 2 * (mass * sums + rest * (sums + rest_sums)) \
            + 2 * E * abs(float(loss[n]))
        w = w * temperature * (1.0 if upstream is None else float(upstream[n]))
        named = torch.zeros(v, dtype=torch.float64).index_add_(0, at, p)
        off = rest / s if s > 0 else 0.0
        grad[n] = w * (q * mass - named - torch.where(beyond, q * off, 0.0))
        own = (3 * arg + 8) * E
        # an exponential below 2^-126 is zero; beside a logit of the row the sum of all is 1 at
        # least, so its factor in the gradient is w (mass + off) at most
        grad_e[n] += abs(w) * 2.0 ** -126 * (mass + off)
        grad_e[n] += abs(w) * (q * mass * (own + sums) + named * 6 * E * max(1, len(at) ** 0.5)
                              + torch.where(beyond, q * off * (own + rest_sums), 0.0))
    return loss, loss_e, grad, grad_e
