"""A linear step on MXFP4 operands whose backward would be refused is refused in its forward."""
from __future__ import annotations

import ctypes

import pytest

from conftest import dpa_mod


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1 << 24, 8, 8), (500, 1 << 24, 32), (32, 32, 1 << 24), (0, 8, 8), (8, 0, 8)])
def test_sizes_that_are_taken(m, n, k):
    dpa_mod("mxfp4")._check_products(m, n, k, True, True)


@pytest.mark.parametrize("m,n,k,wanted,what", [
    ((1 << 24) + 32, 8, 8, (False, True), "dweight"), (8, (1 << 24) + 32, 8, (True, False), "dx"), (8, 8, (1 << 24) + 1, (False, False), "output"),
    (513, 1, 32_000_000, (True, False), "output"), (8, 8, 1 << 25, (True, True), "output")])
def test_sizes_that_are_refused(m, n, k, wanted, what):
    check = dpa_mod("mxfp4")._check_products
    with pytest.raises(ValueError, match=f"the product of {what}, .* is beyond"):
        check(m, n, k, *wanted)
    if what != "output":        # taken where that gradient is not wanted
        check(m, n, k, False, False)


@pytest.mark.parametrize("cols", [(1 << 30) - 63, (1 << 30) - 1, 1 << 30])
def test_column_sums_of_more_workgroups_than_a_launch_has(cols):
    """64 columns to a workgroup of 256: beyond 2^24 - 1 of them their number would wrap."""
    lib = dpa_mod("_lib").load()
    fake = ctypes.c_void_p(0x1000)      # never dereferenced
    assert lib.dpa_column_sum(fake, 0, 4, cols, cols, fake, fake, 1 << 40, None) == -2
