"""Workspaces of the norms' and the embedding's gradients, from the smallest sizes to the largest."""

import pytest

from mfattn import _lib

L = _lib.LIB


@pytest.mark.parametrize("dtype", [_lib.DTYPE_F32, _lib.DTYPE_BF16])
def test_norm_workspace_holds_every_workgroup(dtype):
    for rows in (1, 2, 63, 64, 1000, 1024, 1025, 32768, 1 << 22):
        for dim in (1, 7, 64, 771, 1024, 2048, 2056, 8192, 16384):
            n = L.mf_norm_bwd_workspace_bytes(rows, dim, dtype)
            # pairs of rows of dim floats: one a workgroup, at most 512; none for few rows
            assert n % (8 * dim) == 0 and n // (8 * dim) <= 512
            assert n // (8 * dim) <= max(1, rows)
            assert (n > 0) == (rows > 1024)


def test_embedding_workspace():
    for n in (1, 64, 8192, 8193, 40000, 1 << 20, 1 << 24):
        for d in (1, 72, 1024):
            last = 0
            for v in (1, 511, 512, 65536, 1 << 18, 1 << 27):
                got = L.mf_embed_bwd_workspace_bytes(n, v, d)
                # two lists of the tokens at least, and fp32 pieces of at most a quarter of them
                assert got >= 16 * n
                assert got <= 16 * n + (n // 8 + 1) * 2 * 4 * (d + 4) + (1 << 18)
                assert got >= last
                last = got
    assert L.mf_embed_bwd_workspace_bytes(1 << 24, 4, 1 << 10) > 0
    assert L.mf_embed_bwd_workspace_bytes(1 << 24, 4, (1 << 10) + 1) == 0


def test_distillation_stats():
    for rows, top in ((1, 1), (4096, 64), (1 << 21, 1024)):
        assert L.mf_distill_stats_bytes(rows, top) == 4 * rows * (4 + top)
