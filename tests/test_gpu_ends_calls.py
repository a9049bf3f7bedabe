"""Ways to call the norms, the embedding and the distillation loss that their documentation allows:
in place through the C ABI, from several threads, under checkpointing, past their limits."""

import threading

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

from mfattn import _lib
from mfattn.kernels import distillation, embedding, normalization

pytestmark = pytest.mark.gpu

L = _lib.LIB


def _stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("center", [1, 0], ids=["layer", "rms"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [5, 64, 100, 771, 1024, 2047, 4096, 5001, 16384])
@pytest.mark.parametrize("rows", [67, 1024, 1500])
def test_norms_in_place(rows, d, dtype, center, device):
    code = _lib.DTYPE_BF16 if dtype is torch.bfloat16 else _lib.DTYPE_F32
    g = torch.Generator(device=device).manual_seed(d)
    x, dy = (torch.randn(rows, d, generator=g, device=device).to(dtype) for _ in range(2))
    w = torch.randn(d, generator=g, device=device).to(dtype)
    y, dx, stats = torch.empty_like(x), torch.empty_like(x), torch.empty(rows, 2, device=device)
    dw, ws = torch.empty_like(w), torch.empty(L.mf_norm_bwd_workspace_bytes(rows, d, code),
                                              dtype=torch.uint8, device=device)

    def forward(x, y):
        _lib.check(L.mf_norm(x.data_ptr(), d, w.data_ptr(), None, code, code, rows, d, center, 1e-5,
                             y.data_ptr(), stats.data_ptr(), _stream()))

    def backward(dy, dx):
        _lib.check(L.mf_norm_bwd(x.data_ptr(), d, w.data_ptr(), stats.data_ptr(), dy.data_ptr(), d,
                                 code, code, rows, d, center, dx.data_ptr(), dw.data_ptr(), None,
                                 ws.data_ptr(), ws.numel(), _stream()))

    forward(x, y)
    backward(dy, dx)
    first = dw.clone()
    backward(dy, dy)
    assert torch.equal(dy, dx) and torch.equal(first, dw)
    forward(x, x)
    assert torch.equal(x, y)


def test_limits_are_errors_with_the_librarys_message(device):
    f = torch.zeros
    for call, text in (
            (lambda: normalization.layer_norm(f(2, 16385, device=device), f(16385, device=device)),
             "at most"),
            (lambda: embedding.embed(f(3, dtype=torch.int64, device=device),
                                     f(2, 65537, device=device)), "at most"),
            (lambda: embedding.embed(f(3, dtype=torch.int64, device=device),
                                     f(2, 8, device=device), scale=1e39), "scale must be finite"),
            (lambda: distillation.top_logits_loss(f(1, 2000, device=device), f(1, 1025, device=device),
                                                  f(1, 1025, dtype=torch.int32, device=device)),
             "at most"),
            (lambda: distillation.top_logits_loss_and_gradient(
                f(1, 393217, device=device), f(1, 5, device=device),
                f(1, 5, dtype=torch.int32, device=device)), "at most")):
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(_lib.MfValueError, match=text) as e:
                call()
            assert e.value.code in (_lib.ERR_SHAPE, _lib.ERR_INVALID_ARGUMENT)
    with pytest.raises(_lib.MfValueError, match="at most"):  # and where a graph is recorded
        normalization.rms_norm(f(1, 16385, device=device, requires_grad=True), f(16385, device=device))
    # the same thread goes on
    assert normalization.rms_norm(torch.ones(1, 4, device=device), torch.ones(4, device=device)).sum() > 3.9


def test_parameters_at_odd_offsets(device):
    flat = torch.randn(4000, device=device).bfloat16()
    x = torch.randn(9, 1001, device=device).bfloat16()
    w, b = flat[1:1002], flat[1501:2502]
    assert torch.equal(normalization.layer_norm(x, w, b), normalization.layer_norm(x, w.clone(), b.clone()))
    wide = torch.randn(9, 1030, device=device).bfloat16()
    for params in (flat, flat.float()):
        got = normalization.rms_norm(wide[:, 7:1008], params[3:1004])
        assert torch.equal(got, normalization.rms_norm(wide[:, 7:1008].clone(), params[3:1004].clone()))


def _losses(device, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    table = torch.randn(700, 256, generator=g, device=device).requires_grad_()
    w = torch.randn(256, generator=g, device=device).requires_grad_()
    ids = torch.randint(0, 700, (90,), generator=g, device=device)
    tids = torch.rand(90, 700, generator=g, device=device).argsort(1)[:, :7].contiguous()
    t = torch.randn(90, 7, generator=g, device=device)

    def head(x, w, table):
        return distillation.top_logits_loss(normalization.rms_norm(x, w) @ table.t(), t, tids,
                                            temperature=3.0)

    return table, w, ids, head


def test_checkpointed_layers(device):
    table, w, ids, head = _losses(device, 1)
    x = embedding.embed(ids, table, scale=2.0)
    want = torch.autograd.grad(head(x, w, table).sum(), (table, w))
    x = embedding.embed(ids, table, scale=2.0)
    loss = checkpoint(head, x, w, table, use_reentrant=False)
    got = torch.autograd.grad(loss.sum(), (table, w))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_several_threads_at_once(device):
    want, got = {}, {}

    def work(k, to, rounds):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(rounds):
                table, w, ids, head = _losses(device, k)
                loss = head(embedding.embed(ids, table), w, table)
                to[k] = (loss.detach(), *torch.autograd.grad(loss.sum(), (table, w)))
            torch.cuda.current_stream().synchronize()

    for k in range(4):
        work(k, want, 1)
    threads = [threading.Thread(target=work, args=(k, got, 12)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(4):
        for a, b in zip(got[k], want[k]):
            assert torch.equal(a, b)


def test_the_operands_may_not_change_before_the_backward_pass(device):
    x = torch.randn(4, 64, device=device)
    w = torch.ones(64, device=device, requires_grad=True)
    y = normalization.rms_norm(x, w)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    z = torch.randn(4, 64, device=device, requires_grad=True)
    held = z * 1
    t, tids = torch.zeros(4, 2, device=device), torch.tensor([[1, 2]] * 4, device=device)
    loss = distillation.top_logits_loss(held, t, tids)
    with torch.no_grad():
        distillation.top_logits_loss_and_gradient(held, t, tids, out=held)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()


def test_a_graph_walked_twice(device):
    table, w, ids, head = _losses(device, 2)
    loss = head(embedding.embed(ids, table), w, table).sum()
    first = torch.autograd.grad(loss, (table, w), retain_graph=True)
    second = torch.autograd.grad(loss, (table, w))
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_tensors_on_the_host_beside_device_tensors(device):
    x = torch.ones(2, 8, device=device)
    with pytest.raises(ValueError, match="GPU only"):
        normalization.rms_norm(x, torch.ones(8))
    with pytest.raises(ValueError, match="GPU only"):
        embedding.embed(torch.zeros(3, dtype=torch.int64), x)
    with pytest.raises(ValueError, match="GPU only"):
        distillation.top_logits_loss(x, torch.ones(2, 3), torch.zeros(2, 3, dtype=torch.int64, device=device))


def test_function_transforms_are_refused(device):
    x = torch.randn(3, 4, 32, device=device)
    w = torch.randn(32, device=device)
    ids = torch.randint(0, 32, (3, 4, 5), device=device)
    t = torch.randn(3, 4, 5, device=device)
    for call in (lambda x: normalization.layer_norm(x, w).sum(),
                 lambda x: embedding.embed(ids[0], x[0]).sum(),
                 lambda x: distillation.top_logits_loss(x[0], t[0], ids[0]).sum()):
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.grad(call)(x)
    for call in (lambda x: normalization.layer_norm(x, w),
                 lambda x: embedding.embed(ids[0], x),
                 lambda x: distillation.top_logits_loss(x, t[0], ids[0])):
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.vmap(call)(x)
    # nothing was launched on the way, and eager calls go on
    torch.cuda.synchronize()
    assert normalization.layer_norm(x, w).shape == x.shape


def test_inference_mode(device):
    x, w = torch.randn(5, 64, device=device), torch.randn(64, device=device)
    ids, t = torch.randint(0, 64, (5, 3), device=device), torch.randn(5, 3, device=device)
    y = normalization.layer_norm(x, w)
    e = embedding.embed(ids, torch.stack([w] * 64))
    alone = distillation.top_logits_loss(x, t, ids)
    loss, grad = distillation.top_logits_loss_and_gradient(x, t, ids)
    with torch.inference_mode():
        assert torch.equal(normalization.layer_norm(x, w), y)
        assert torch.equal(embedding.embed(ids, torch.stack([w] * 64)), e)
        assert torch.equal(distillation.top_logits_loss(x, t, ids), alone)
        mine = x.clone()
        assert torch.equal(distillation.top_logits_loss_and_gradient(mine, t, ids, out=mine)[0], loss)
        assert torch.equal(mine, grad)


def _wrong_calls(device):
    f = lambda *shape, **kw: torch.zeros(*shape, device=device, **kw)  # noqa: E731
    half, brain = torch.float16, torch.bfloat16
    norm, rms = normalization.layer_norm, normalization.rms_norm
    x, w, g = f(3, 8), f(8), f(8, requires_grad=True)
    yield "weight", lambda: norm(x, f(9))
    yield "D", lambda: norm(f(()), w)
    yield "D", lambda: rms(f(3, 0), f(0))
    yield "weight", lambda: norm(x, f(8, 1))
    yield "weight", lambda: norm(x, f(8, dtype=brain))
    yield "bias", lambda: norm(x, w, f(7))
    yield "bias", lambda: norm(x.bfloat16(), w, f(8, dtype=brain))
    yield "dtype", lambda: norm(x.to(half), w.to(half))
    yield "dtype", lambda: norm(x.double(), w)
    yield "eps", lambda: norm(x, w, eps=float("nan"))
    yield "eps", lambda: rms(x, w, eps=-1e-9)
    yield "eps", lambda: rms(x, w, eps=float("inf"))
    ids, table = f(4, dtype=torch.int64), f(5, 8)
    yield "table", lambda: embedding.embed(ids, w)
    yield "table", lambda: embedding.embed(ids, f(0, 8))
    yield "integers", lambda: embedding.embed(f(4), table)
    yield "integers", lambda: embedding.embed(f(4, dtype=torch.bool), table)
    yield "scale", lambda: embedding.embed(ids, table, scale=float("inf"))
    yield "padding", lambda: embedding.embed(ids, table, padding_id=1 << 63)
    yield "dtype", lambda: embedding.embed(ids, table.to(half))
    z, t, k, n = f(3, 8), f(3, 2), f(3, 2, dtype=torch.int32), f(3)
    loss = distillation.top_logits_loss
    yield "teacher", lambda: loss(z, f(3, 3), k)
    yield "teacher", lambda: loss(z, f(2, 2), f(2, 2, dtype=torch.int32))
    yield "teacher", lambda: loss(z, f(3, 0), f(3, 0, dtype=torch.int32))
    yield "teacher", lambda: loss(z, t[0], k[0])
    yield "integers", lambda: loss(z, t, t)
    yield "logits", lambda: loss(f(3, 0), t, k)
    yield "dtype", lambda: loss(z.to(half), t, k)
    yield "dtype", lambda: loss(z, t.to(half), k)
    yield "teacher_total", lambda: loss(z, t, k, teacher_total=f(3, 1))
    yield "weights", lambda: loss(z, t, k, weights=f(1))
    yield "weights", lambda: loss(z, t, k, weights=f(3, dtype=torch.int32))
    yield "temperature", lambda: loss(z, t, k, temperature=0.0)
    yield "temperature", lambda: loss(z, t, k, temperature=2e6)
    yield "detach", lambda: loss(z, t.clone().requires_grad_(), k)
    yield "detach", lambda: loss(z, t, k, weights=n.clone().requires_grad_())
    both = distillation.top_logits_loss_and_gradient
    yield "records no graph", lambda: both(z.clone().requires_grad_(), t, k)
    yield "teacher", lambda: both(z, f(3, 3), k)
    yield "temperature", lambda: both(z, t, k, temperature=float("nan"))
    yield "at most", lambda: both(z, f(3, 1025), f(3, 1025, dtype=torch.int32))

    def dual(call, x):
        with forward_ad.dual_level():
            call(forward_ad.make_dual(x, torch.ones_like(x)))

    yield "tangent", lambda: dual(lambda x: norm(x, g), x)
    yield "tangent", lambda: dual(lambda w: norm(x, w), w)
    yield "tangent", lambda: dual(lambda b: norm(x, w, b), w)
    yield "tangent", lambda: dual(lambda table: embedding.embed(ids, table), table)
    yield "tangent", lambda: dual(lambda z: loss(z, t, k), z)
    yield "tangent", lambda: dual(lambda n: loss(z, t, k, weights=n), n)


def test_wrong_device_tensors_are_refused(device):
    for text, call in _wrong_calls(device):
        with pytest.raises(ValueError, match=text):
            call()


def test_operands_of_another_kind_give_the_same(device):
    g = torch.Generator(device=device).manual_seed(5)
    x = torch.randn(6, 40, generator=g, device=device)
    w = torch.randn(40, generator=g, device=device)
    # parameters that are not dense, and an integer for eps
    y = normalization.layer_norm(x, w, w, eps=1.0)
    apart = torch.stack([w, w], 1)[:, 0]
    assert not apart.is_contiguous()
    assert torch.equal(normalization.layer_norm(x, apart, apart, eps=1), y)
    assert torch.equal(normalization.layer_norm(x.t().contiguous().t(), w, w, eps=1.0), y)
    ids = torch.randint(0, 6, (4, 7), generator=g, device=device)
    e = embedding.embed(ids, x, scale=2.0, padding_id=3)
    assert torch.equal(embedding.embed(ids.t().contiguous().t(), x, scale=2, padding_id=3), e)
    assert torch.equal(embedding.embed(ids.to(torch.int16), x.t().contiguous().t(), scale=2.0, padding_id=3), e)
    t, k = torch.randn(6, 5, generator=g, device=device), ids[:1, :5].expand(6, 5)
    n = torch.rand(6, generator=g, device=device)
    loss = distillation.top_logits_loss(x, t, k.contiguous(), weights=n, temperature=2.0)
    for other in (dict(weights=n.double()), dict(weights=torch.stack([n, n], 1)[:, 1]), dict(temperature=2)):
        assert torch.equal(distillation.top_logits_loss(x, t, k, **{"weights": n, "temperature": 2.0, **other}),
                           loss)
    pair = distillation.top_logits_loss_and_gradient(x, t, k.contiguous(), weights=n, temperature=2.0)
    for other in (dict(weights=n.double()), dict(temperature=2), dict(out=torch.empty_like(x))):
        more = {"weights": n, "temperature": 2.0, **other}
        for a, b in zip(distillation.top_logits_loss_and_gradient(x, t, k, **more), pair):
            assert torch.equal(a, b) and not a.requires_grad
    with torch.no_grad():  # nothing is recorded: a teacher may require what it likes
        assert torch.equal(distillation.top_logits_loss(x, t.clone().requires_grad_(), k, weights=n,
                                                        temperature=2.0), loss)


def _steps(device):
    g = torch.Generator(device=device).manual_seed(11)
    x = torch.randn(6, 40, generator=g, device=device).requires_grad_()
    w = torch.randn(40, generator=g, device=device).requires_grad_()
    ids = torch.randint(0, 6, (9, 4), generator=g, device=device)
    t, k = torch.randn(6, 4, generator=g, device=device), ids[:6].to(torch.int32)
    n = torch.rand(6, generator=g, device=device)
    return ((lambda: normalization.layer_norm(x, w, w), (x, w)), (lambda: embedding.embed(ids, x), (x,)),
            (lambda: distillation.top_logits_loss(x, t, k, weights=n), (x,)))


def _across(t):
    """The same values, strides the other way round."""
    return t if t.dim() < 2 else t.transpose(-1, -2).contiguous().transpose(-1, -2)


@pytest.mark.parametrize("how", ["host", "strides"])
def test_saved_tensors_that_were_elsewhere(how, device):
    hooks = (torch.autograd.graph.save_on_cpu() if how == "host" else
             torch.autograd.graph.saved_tensors_hooks(lambda t: t, _across))
    for call, leaves in _steps(device):
        want = torch.autograd.grad(call().sum(), leaves)
        with hooks:
            out = call()
        for a, b in zip(torch.autograd.grad(out.sum(), leaves), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("other", [lambda t: t.cpu(), lambda t: t.half(), lambda t: t[:-1],
                                   lambda t: torch.cat([t, t])], ids=["host", "half", "less", "more"])
def test_saved_tensors_that_come_back_changed(other, device):
    for call, leaves in _steps(device):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other):
            out = call()
        with pytest.raises(RuntimeError, match="came back"):
            torch.autograd.grad(out.sum(), leaves)
