"""The C ABI's loss with its gradient and what the backward pass needs in one call."""

import pytest
import torch

import _ends
from mfattn import _lib

pytestmark = pytest.mark.gpu

L = _lib.LIB


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", [100, 8193, 70001])
@pytest.mark.parametrize("total", [False, True], ids=["softmax", "total"])
def test_stats_beside_the_gradient(v, dtype, total, device):
    rows, k, temperature = 6, 9, 1.5
    g = torch.Generator(device=device).manual_seed(v)
    z = 2 * torch.randn(rows, v, generator=g, device=device)
    ids = torch.rand(rows, v, generator=g, device=device).argsort(1)[:, :k].to(torch.int32).contiguous()
    t = 3 * torch.randn(rows, k, generator=g, device=device)
    z, t = z.to(dtype), t.to(dtype)
    mass = torch.logsumexp(t.float() / temperature, 1) + 0.2 if total else None
    weights = torch.rand(rows, generator=g, device=device)
    weights[1] = 0
    up = torch.linspace(-1, 2, rows, device=device)
    code = _lib.DTYPE_BF16 if dtype is torch.bfloat16 else _lib.DTYPE_F32
    loss = torch.empty(rows, device=device)
    stats = torch.full((rows * (4 + k),), float("nan"), device=device)
    grad, back = torch.empty_like(z), torch.empty_like(z)
    stream = torch.cuda.current_stream().cuda_stream
    total_at = mass.data_ptr() if total else None
    _lib.check(L.mf_distill(z.data_ptr(), v, t.data_ptr(), code, ids.data_ptr(), 4, total_at,
                            weights.data_ptr(), code, rows, v, k, temperature, loss.data_ptr(),
                            stats.data_ptr(), 4 * stats.numel(), grad.data_ptr(), v, stream))
    _lib.check(L.mf_distill_bwd(z.data_ptr(), v, ids.data_ptr(), 4, weights.data_ptr(),
                                stats.data_ptr(), 4 * stats.numel(), up.data_ptr(), code, rows, v, k,
                                temperature, back.data_ptr(), v, stream))
    want = _ends.distill(z, t, ids, temperature, mass, weights)
    _ends.check(loss, *want[:2], "loss")
    _ends.check(grad, *want[2:], "gradient")
    want = _ends.distill(z, t, ids, temperature, mass, weights, up)
    _ends.check(back, *want[2:], "gradient from the stats")
