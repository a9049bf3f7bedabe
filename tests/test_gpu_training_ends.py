"""A packed training step from tokens to loss and back to the table, and captured steps."""

import pytest
import torch

from mfattn.kernels import attention, distillation, embedding, normalization, prologue

pytestmark = pytest.mark.gpu

D, HQ, HKV, V, T, B = 256, 4, 2, 611, 96, 2


def _batch(device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    ids = torch.randint(0, V, (B, T), generator=g, device=device)
    seg = torch.ones(B, T, dtype=torch.int32, device=device)
    seg[:, 40:] = 2
    seg[:, 80:] = 0
    ids = ids.masked_fill(seg == 0, -1)
    top = torch.rand(B, T, V, generator=g, device=device).topk(6, -1)
    weights = (seg != 0).float() / (seg != 0).sum()
    return ids, seg, 5 * top.values, top.indices, weights


def _params(device, dtype):
    g = torch.Generator(device=device).manual_seed(3)

    def normal(*shape, scale):
        return (scale * torch.randn(*shape, generator=g, device=device)).to(dtype).requires_grad_()

    return {"table": normal(V, D, scale=0.2), "first": normal(D, scale=1.0),
            "qkv": normal(D, (HQ + 2 * HKV) * 64, scale=D ** -0.5),
            "q_gain": normal(64, scale=1.0), "k_gain": normal(64, scale=1.0),
            "back": normal(HQ * 64, D, scale=0.06),
            "last": normal(D, scale=1.0), "bias": normal(D, scale=0.1)}


def _step(p, batch):
    ids, seg, teacher, tids, weights = batch
    x = embedding.embed(ids, p["table"], scale=D ** 0.5)
    h = normalization.rms_norm(x, p["first"])
    q, k, v = (h @ p["qkv"]).split((HQ * 64, HKV * 64, HKV * 64), -1)
    q, k, v = (t.unflatten(-1, (-1, 64)) for t in (q, k, v))
    q, k = prologue.qk_norm_rope(q, k, p["q_gain"], p["k_gain"], prologue.segment_positions(seg),
                                 eps=1e-5, rope_theta=1e4)
    a = attention.packed_causal_attention(q, k, v, (seg != 0).int(), seg, backend="hip")
    y = normalization.layer_norm(x + a.flatten(2) @ p["back"], p["last"], p["bias"])
    logits = y @ p["table"].t()
    return distillation.top_logits_loss(logits, teacher, tids, temperature=2.0, weights=weights)


def _reference(p, batch):
    """The same step in float64 on the CPU, by torch."""
    ids, seg, teacher, tids, weights = (t.cpu() for t in batch)
    p = {n: t.detach().cpu().double().requires_grad_() for n, t in p.items()}
    real = ids >= 0
    x = torch.where(real[..., None], p["table"][ids.clamp(min=0)], 0) * D ** 0.5

    def rms(t, w):
        return t * ((t * t).mean(-1, keepdim=True) + 1e-5) ** -0.5 * w

    q, k, v = (rms(x, p["first"]) @ p["qkv"]).split((HQ * 64, HKV * 64, HKV * 64), -1)
    q, k, v = (t.unflatten(-1, (-1, 64)) for t in (q, k, v))
    pos = torch.where(seg == 1, torch.arange(T), torch.arange(T) - 40) * (seg != 0)
    angle = pos[..., None].double() * 1e4 ** (-torch.arange(32).double() / 32)
    c, s = (torch.cat((f(angle),) * 2, -1)[:, :, None] for f in (torch.cos, torch.sin))

    def turn(t):
        return t * c + torch.cat((-t[..., 32:], t[..., :32]), -1) * s

    q, k = turn(rms(q, p["q_gain"])), turn(rms(k, p["k_gain"]))
    k, v = (t.repeat_interleave(HQ // HKV, 2) for t in (k, v))
    scores = (q.transpose(1, 2) @ k.transpose(1, 2).transpose(2, 3).contiguous()) / 8
    seen = (seg[:, :, None] == seg[:, None]) & (seg != 0)[:, None] & torch.ones(T, T).tril().bool()
    w = scores.masked_fill(~seen[:, None], -1e300).softmax(-1) * seen.any(-1)[:, None, :, None]
    a = (w @ v.transpose(1, 2)).transpose(1, 2).flatten(2)
    y = x + a @ p["back"]
    y = y - y.mean(-1, keepdim=True)
    y = rms(y, p["last"]) + p["bias"]
    logq = (y @ p["table"].t() / 2).log_softmax(-1).gather(-1, tids)
    t = teacher.double() / 2
    logt = t.log_softmax(-1)
    loss = 4 * (logt.exp() * (logt - logq)).sum(-1) * weights.double()
    return loss, p


def test_a_packed_step_from_tokens_to_loss(device):
    p, batch = _params(device, torch.float32), _batch(device)
    loss = _step(p, batch)
    loss.sum().backward()
    want, ref = _reference(p, batch)
    want.sum().backward()
    # float32 through nine operators: each adds a few roundings of sums over at most 611 terms,
    # (611 + 30) * 2^-24 of the sums of sizes at worst, typically their root; products of nine
    # such factors, times the growth of sums of sizes over sums (below 10 here each)
    room = 9 * 641 * 2.0 ** -24 * 10
    assert (loss.detach().cpu().double() - want.detach()).norm() <= room * want.detach().norm()
    for name, t in p.items():
        g, r = t.grad.cpu().double(), ref[name].grad
        assert (g - r).norm() <= room * r.norm(), name
    assert not loss[:, 80:].any()


def test_a_step_captured_and_replayed(device):
    """New tokens, tables and teachers in the same buffers; eager work between the replays."""
    dtype = torch.bfloat16
    side = torch.cuda.Stream()
    p, batch = _params(device, dtype), _batch(device)
    names = list(p)

    def step():
        loss = _step(p, batch)
        return (loss.detach(), *torch.autograd.grad(loss.sum(), [p[n] for n in names]))

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (5, 6, 7):
        for t, new in zip(batch, _batch(device, seed)):
            t.copy_(new)
        with torch.no_grad():
            p["table"].copy_(torch.randn(V, D, device=device) * 0.1 * seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        # library products in the graph and outside of it may take other kernels: the norms,
        # the lookup and the loss see their results
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# launches of few rows and tokens, and of many
SIZES = [(300, 2000, 40), (1500, 9001, 600)]


def _each(device, rows, tokens, logits):
    """Every operator's pass over buffers that the caller refills."""
    x = torch.randn(rows, 1024, device=device).bfloat16()
    w = torch.randn(1024, device=device).bfloat16().requires_grad_()
    dy = torch.randn(rows, 1024, device=device).bfloat16()
    ids = torch.randint(0, 3000, (tokens,), device=device)
    table = torch.randn(3000, 136, device=device).requires_grad_()
    dout = torch.randn(tokens, 136, device=device)
    z = torch.randn(logits, 9001, device=device).bfloat16().requires_grad_()
    t, tids = torch.randn(logits, 16, device=device), torch.randint(0, 9001, (logits, 16), device=device)
    total = torch.logsumexp(t, 1) + 0.1
    leaf = x.requires_grad_()

    def one():
        return torch.autograd.grad(normalization.layer_norm(leaf, w, w.detach()), (leaf, w), dy)

    def two():
        return torch.autograd.grad(embedding.embed(ids, table), table, dout)

    def three():
        loss = distillation.top_logits_loss(z, t, tids, teacher_total=total)
        with torch.no_grad():
            both = distillation.top_logits_loss_and_gradient(z, t, tids, teacher_total=total)
        return (loss.detach(), *torch.autograd.grad(loss.sum(), z), *both)

    def refill():
        with torch.no_grad():
            for b in (x, dy, dout, z, t):
                b.normal_()
            ids.copy_(torch.randint(0, 3000, (tokens,), device=device))
            tids.copy_(torch.randint(0, 9001, (logits, 16), device=device))
            total.copy_(torch.logsumexp(t, 1) + 0.2)

    return (one, two, three), refill


@pytest.mark.parametrize("sizes", SIZES)
def test_two_graphs_over_the_same_operands(sizes, device):
    """Captured one by one, replayed in turn several times: no graph lives on another's scratch."""
    calls, refill = _each(device, *sizes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in calls:
            c()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for c in (*calls, *calls):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = c()
        graphs.append((g, out))
    for _ in range(3):
        refill()
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in out] for _, out in graphs]
        want = [c() for c in calls]
        torch.cuda.synchronize()
        for i, out in enumerate(got):
            for a, b in zip(out, want[i % 3]):
                assert torch.equal(a, b), i


@pytest.mark.parametrize("sizes", SIZES)
def test_calls_in_flight_on_two_streams(sizes, device):
    first, _ = _each(device, *sizes)
    second, refill = _each(device, *sizes)
    want = [[c() for c in calls] for calls in (first, second)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        got = [[], []]
        for i in range(3):
            for k, calls in enumerate((first, second)):
                with torch.cuda.stream(streams[k]):
                    got[k].append(calls[i]())
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            for s, t in zip(x, y):
                assert torch.equal(s, t)
