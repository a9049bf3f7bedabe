"""Refusals of operands that are not there, one by one (no GPU needed)."""

import pytest

from mfattn import _lib

L = _lib.LIB
P = 1 << 20  # an address that no refused call reads


@pytest.mark.parametrize("gone", ["ids", "table", "out"])
def test_lookup(gone):
    a = {name: P for name in ("ids", "table", "out")}
    a[gone] = None
    assert L.mf_embed(a["ids"], 8, a["table"], 64, 1, 4, 10, 64, -1, 1.0, a["out"],
                      None) == _lib.ERR_INVALID_ARGUMENT
    assert "non-null" in L.mf_last_error().decode()


@pytest.mark.parametrize("gone", ["ids", "dout", "dtable"])
def test_lookup_gradient(gone):
    a = {name: P for name in ("ids", "dout", "dtable")}
    a[gone] = None
    assert L.mf_embed_bwd(a["ids"], 8, a["dout"], 64, 1, 4, 10, 64, -1, 1.0, a["dtable"], P, 1 << 30,
                          None) == _lib.ERR_INVALID_ARGUMENT
    assert "non-null" in L.mf_last_error().decode()
