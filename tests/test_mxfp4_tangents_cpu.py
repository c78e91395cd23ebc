"""Where the MXFP4 operators have no gradient they refuse tensors with a forward-mode tangent instead of dropping it."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from conftest import dpa_mod


@pytest.mark.parametrize("grad", [True, False])
def test_queries_with_a_tangent_are_refused(grad):
    M = dpa_mod("mxfp4")
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    q = torch.zeros((1, 3, 2, 64))
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(ValueError, match="no gradient"):
            M.cross_attention_mxfp4(dual, M.MXFP4(u8(1, 5, 2, 2, 32), u8(1, 5, 2, 2, 2)))


@pytest.mark.parametrize("which", ["x", "bias"])
def test_an_operand_as_weight_and_a_tangent(which):
    M = dpa_mod("mxfp4")
    w = M.MXFP4Operand(torch.zeros(64, dtype=torch.uint8), 4, 32)
    x, bias = torch.zeros((3, 32)), torch.zeros(4)
    with forward_ad.dual_level():
        if which == "x":
            x = forward_ad.make_dual(x, torch.ones_like(x))
        else:
            bias = forward_ad.make_dual(bias, torch.ones_like(bias))
        with pytest.raises(ValueError, match="need the weight itself"):
            M.linear_mxfp4(x, w, bias)
