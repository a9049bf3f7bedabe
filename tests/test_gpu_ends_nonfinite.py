"""Values that are not finite stay where the definitions put them."""

import pytest
import torch

from mfattn.kernels import embedding, normalization

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]
VALUES = [float("nan"), float("inf"), -float("inf")]


# every number of lanes and vectors a row, odd widths, few rows and many
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [3, 64, 100, 512, 771, 1024, 2048, 4096, 5001, 16384])
@pytest.mark.parametrize("rows", [40, 1500])
@pytest.mark.parametrize("center", [True, False], ids=["layer", "rms"])
def test_norm_gradients_beside_a_row_that_is_not_finite(center, rows, d, dtype, device):
    g = torch.Generator(device=device).manual_seed(d + rows)
    x, dy = (torch.randn(rows, d, generator=g, device=device).to(dtype) for _ in range(2))
    w, b = (torch.randn(d, generator=g, device=device).to(dtype) for _ in range(2))

    def all_of(x, dy):
        leaves = [t.clone().requires_grad_() for t in ((x, w, b) if center else (x, w))]
        y = normalization.layer_norm(*leaves) if center else normalization.rms_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    clean = all_of(x, dy)
    for row, col in ((7, d // 2), (rows - 1, d - 1)):
        keep = torch.arange(rows, device=device) != row
        for value in VALUES:
            bad = x.clone()
            bad[row, col] = value
            y, dx, *dp = all_of(bad, dy)
            assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
            assert y[row].isnan().any() and dx[row].isnan().any()
            assert dp[0].isnan().any()
            if center:  # (the bias knows dy alone)
                assert torch.equal(dp[1], clean[3])
            if value != value:
                assert y[row].isnan().all() and dx[row].isnan().all() and dp[0].isnan().all()
            bad = dy.clone()
            bad[row, col] = value
            y, dx, *dp = all_of(x, bad)
            assert torch.equal(y, clean[0]) and torch.equal(dx[keep], clean[1][keep])
            assert dx[row].isnan().any()
            for p, q in zip(dp, clean[2:]):
                assert not p[col].isfinite() and torch.equal(p[:col], q[:col]) and torch.equal(
                    p[col + 1:], q[col + 1:])
                if value != value:
                    assert p[col].isnan()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [3, 64, 129, 1024, 2056])
def test_embedding_rows_that_are_not_finite(d, dtype, device):
    """Tokens without a row get zeros, whatever the rows hold that stand in for theirs; a token's
    gradient is its own id's."""
    for row in (0, 4, 20):
        for value in VALUES:
            table = torch.randn(21, d, device=device).to(dtype)
            table[row] = value
            ids = torch.tensor([-1, 21, 1 << 40, 5, 3, -(1 << 50), row, 5], device=device)
            out = embedding.embed(ids, table, scale=2.0, padding_id=3)
            assert not out[[0, 1, 2, 4, 5]].any()
            assert torch.equal(out[[3, 7]], (table[[5, 5]].float() * 2).to(dtype))
            assert torch.equal(out[6].isnan(), table[row].isnan())
            assert torch.equal(out[6].isinf(), table[row].isinf())
            out = embedding.embed(ids, table, padding_id=row)
            assert not out[[0, 1, 2, 5, 6]].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [3, 129, 1024])
@pytest.mark.parametrize("n", [50, 1500, 9000, 40000])
def test_embedding_gradients_that_are_not_finite(n, d, dtype, device):
    g = torch.Generator(device=device).manual_seed(n + d)
    ids = torch.randint(0, 30, (n,), generator=g, device=device)
    ids[::5] = -1
    ids[3] = 17
    dout = torch.randn(n, d, generator=g, device=device).to(dtype)
    leaf = torch.zeros(31, d, device=device, dtype=dtype).requires_grad_()
    (clean,) = torch.autograd.grad(embedding.embed(ids, leaf, padding_id=4), leaf, dout)
    dout[ids == 4] = float("nan")
    dout[::5] = float("inf")
    (got,) = torch.autograd.grad(embedding.embed(ids, leaf, padding_id=4), leaf, dout)
    assert torch.equal(got, clean)
    for value in VALUES:
        dout[3, d - 1] = value
        (got,) = torch.autograd.grad(embedding.embed(ids, leaf, padding_id=4), leaf, dout)
        keep = torch.arange(31, device=device) != 17
        assert torch.equal(got[keep], clean[keep]) and torch.equal(got[17, :-1], clean[17, :-1])
        if value != value:
            assert got[17, -1].isnan()
        else:
            assert got[17, -1] == value
