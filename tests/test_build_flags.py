"""Flags of sources whose operands may hold NaN."""

import pytest

from mfattn import build


@pytest.mark.parametrize("name", ["mf_norm", "mf_embed", "mf_distill"])
def test_values_that_are_not_numbers_are_honoured(name):
    source = build.CSRC / f"{name}.hip"
    assert source.exists()
    assert "-fno-honor-nans" not in build._flags(source)
