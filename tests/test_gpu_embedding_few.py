"""The embedding's gradient of few tokens: around the sizes at which one launch takes it, of whole
numbers, exact in float32 in any order."""

import pytest
import torch

from _helpers import say
from mfattn import _lib
from mfattn.kernels import embedding

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]


def _check(ids, v, dout, scale=1.0, padding=None):
    d = dout.shape[-1]
    leaf = torch.full((v, d), float("nan"), device=dout.device, dtype=dout.dtype).requires_grad_()
    (got,) = torch.autograd.grad(embedding.embed(ids, leaf, scale=scale, padding_id=padding), leaf, dout)
    flat, rows = ids.reshape(-1).long().cpu(), dout.reshape(-1, d).double().cpu()
    real = (flat >= 0) & (flat < v) & (flat != (-1 if padding is None else padding))
    want = torch.zeros(v, d, dtype=torch.float64).index_add_(0, flat[real], rows[real]) * scale
    assert torch.equal(got.cpu(), want.to(dout.dtype))
    return got


def _operands(n, v, d, dtype, device, skew=3):
    g = torch.Generator(device=device).manual_seed(n + 7 * v + d)
    u = torch.rand(n, generator=g, device=device, dtype=torch.float64)
    ids = (v * u ** skew).long().clamp(max=v - 1)
    return ids, torch.randint(-3, 4, (n, d), generator=g, device=device).to(dtype)


# one, two, three and four slabs of columns and more, whole and cut vectors, rows of less than one
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 3, 4, 7, 8, 9, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257,
                               384, 385, 512, 513])
@pytest.mark.parametrize("n, v", [(1, 1), (63, 40), (1025, 300), (5001, 1003), (8192, 4096)])
def test_widths(n, v, d, dtype, device):
    say("few", n, v, d, dtype)
    _check(*(lambda ids, dout: (ids, v, dout))(*_operands(n, v, d, dtype, device)), scale=4.0)


# fewer rows than groups, all groups, several rows each, the last that one launch takes and the next
@pytest.mark.parametrize("d", [16, 128, 200, 512])
@pytest.mark.parametrize("v", [1, 2, 7, 127, 128, 129, 255, 256, 257, 511, 512, 513, 4095, 4096, 4097,
                               131071, 131072, 131073])
def test_vocabularies(v, d, device):
    say("few vocabulary", v, d)
    for n in (1, 700, 8191):
        ids, dout = _operands(n, v, d, torch.bfloat16, device, skew=1)
        ids[0], ids[-1] = v - 1, 0
        _check(ids, v, dout)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 511, 512, 513, 1024, 4096, 8191, 8192, 8193])
@pytest.mark.parametrize("share", [0.0, 0.3, 0.9, 1.0])
@pytest.mark.parametrize("d", [40, 129])
def test_an_id_of_many_tokens(d, share, n, device):
    say("few, one id", n, share, d)
    ids, dout = _operands(n, 700, d, torch.float32, device, skew=1)
    ids[torch.rand(n, device=device) < share] = 333
    _check(ids, 700, dout)


def test_tokens_without_a_row_and_kinds_of_ids(device):
    ids, dout = _operands(6000, 900, 100, torch.float32, device)
    ids[::3] = -1
    ids[1::7] = 900
    ids[2::11] = 1 << 40
    ids[5::13] = -(1 << 40)
    first = _check(ids, 900, dout, padding=17)
    assert not first[17].any()
    assert torch.equal(_check(ids.clamp(-5, 2000).int(), 900, dout, padding=17), first)
    assert torch.equal(_check(ids.view(20, 300), 900, dout.view(20, 300, 100), padding=17), first)
    assert not _check(torch.full_like(ids, -1), 900, dout).any()
    # rows that are not dense, at odd offsets, and one row for all
    wide = torch.full((6000, 150), float("nan"), device=device)
    wide[:, 33:133] = dout
    assert torch.equal(_check(ids, 900, wide[:, 33:133], padding=17), first)
    _check(ids, 900, dout[:1].expand(6000, 100))


def test_the_same_bits_every_time_and_what_lies_beside(device):
    n, v, d = 7000, 1003, 129
    ids, _ = _operands(n, v, d, torch.float32, device)
    dout = torch.randn(n, d, device=device)
    lib, need = _lib.LIB, _lib.LIB.mf_embed_bwd_workspace_bytes(n, v, d)
    around = torch.full((v + 8, d), 7.0, device=device)
    out = around.view(-1)[4 * d - (4 * d) % 4:][:v * d]
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    first = None
    for _ in range(5):
        ws.fill_(255)
        out.fill_(float("nan"))
        _lib.check(lib.mf_embed_bwd(ids.data_ptr(), 8, dout.data_ptr(), d, _lib.DTYPE_F32, n, v, d, -1, 1.0,
                                    out.data_ptr(), ws.data_ptr(), need,
                                    torch.cuda.current_stream().cuda_stream))
        first = out.clone() if first is None else first
        assert torch.equal(out, first)
    flat, at = around.view(-1), 4 * d - (4 * d) % 4
    assert (flat[:at] == 7).all() and (flat[at + v * d:] == 7).all()


def test_captured_and_replayed(device):
    table = torch.randn(1003, 129, device=device)
    ids = torch.zeros(5001, dtype=torch.int64, device=device)
    dout = torch.zeros(5001, 129, device=device)
    leaf = table.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(embedding.embed(ids, leaf), leaf, dout)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(embedding.embed(ids, leaf), leaf, dout)
    for seed in range(4):
        more, rows = _operands(5001, 1003, 129, torch.float32, device, skew=1 + seed)
        ids.copy_(more)
        dout.copy_(rows)
        graph.replay()
        assert torch.equal(got, _check(ids, 1003, dout))
