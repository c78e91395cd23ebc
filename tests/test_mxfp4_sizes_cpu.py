"""A linear step on MXFP4 operands whose backward would be refused is refused in its forward."""
from __future__ import annotations

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
