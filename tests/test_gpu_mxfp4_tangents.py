"""No MXFP4 operator drops a forward-mode tangent in silence, and none minds a level of dual tensors that it has none of."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from conftest import dpa_mod

pytestmark = pytest.mark.gpu


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


def test_dual_tensors_are_refused():
    M = dpa_mod("mxfp4")
    x, w, b = torch.randn((40, 64), device="cuda"), torch.randn((32, 64), device="cuda"), torch.randn(32, device="cuda")
    layer = M.LinearMXFP4(64, 32).cuda()
    layer.keep_weight()
    q = torch.randn((1, 3, 2, 32), device="cuda").bfloat16()
    kv = M.quantize_mxfp4(torch.randn((1, 5, 2, 2, 32), device="cuda"))
    kept = M.mxfp4_operand(w)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            for args in ((dual(x), w, b), (x, dual(w), b), (x, w, dual(b)), (dual(x), kept, b), (x, kept, dual(b))):
                with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
                    M.linear_mxfp4(*args)
            with pytest.raises(ValueError, match="no gradient"):
                M.cross_attention_mxfp4(dual(q), kv)
            with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
                torch.func.functional_call(layer, {"weight": dual(layer.weight.detach())}, (x,))
            # without a tangent the calls are what they are
            assert torch.equal(M.linear_mxfp4(x, kept, b), M.linear_mxfp4_fwd(x, w, b))
            assert torch.equal(M.cross_attention_mxfp4(q, kv), M.cross_attention_mxfp4_fwd(q, kv)[0])
