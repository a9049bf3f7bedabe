"""Sizes of a paged step's workspace and plan against what the calls can use (no GPU needed)."""

import pytest

from mfattn import _lib

L = _lib.LIB


def _partial_rows(tokens, hq, hkv, code):
    """Partial rows of a key head at most, counted from the cuts: `shares` per kind cut tiles of 32
    and 256 rows fewer than `shares` times, and a tile cut n times has n + 1 items."""
    pairs = hkv // 2 if code == _lib.DTYPE_BF16 and hkv % 2 == 0 else hkv
    rows = tokens * (hq // hkv)
    total = 0
    for size, shares in ((32, max(512 // pairs, 1)),
                         (256, max(512 // hkv, 1) if code == _lib.DTYPE_BF16 and rows > 32 else 0)):
        total += min(size, rows) * shares + min(rows, size * shares)
    return total


@pytest.mark.parametrize("code", [_lib.DTYPE_BF16, _lib.DTYPE_F32])
@pytest.mark.parametrize("hq, hkv", [(16, 8), (32, 8), (8, 1), (9, 3), (64, 64), (128, 1)])
@pytest.mark.parametrize("sequences, tokens", [(1, 1), (64, 64), (3, 700), (1, 16384), (64, 131072),
                                               (4096, 400000)])
def test_a_workspace_holds_what_is_cut(sequences, tokens, hq, hkv, code):
    need = L.mf_paged_attn_workspace_bytes(sequences, tokens, hq, hkv, code)
    rows = _partial_rows(tokens, hq, hkv, code)
    # (max, sum) and 64 outputs of a row and key head in float32
    assert 0 < need <= rows * hkv * 264 + 256


def test_workspaces_of_long_steps_do_not_grow():
    sizes = [L.mf_paged_attn_workspace_bytes(64, n, 16, 8, _lib.DTYPE_BF16) for n in (20000, 200000, 1 << 22)]
    assert sizes[0] == sizes[1] == sizes[2] < 100 << 20
    # the plan holds a record per token, and tiles and their items
    for n in (200000, 1 << 22):
        tiles = 64 + n * 2 // 256
        assert L.mf_paged_plan_bytes(64, n, 16, 8, _lib.DTYPE_BF16) < 16 * n + 32 * tiles + (1 << 18)
