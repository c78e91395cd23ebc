"""Sizes at the border of what the MXFP4 linear layer takes: a step is refused whole, before its forward."""
from __future__ import annotations

import pytest
import torch

from conftest import dpa_mod

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])      # (the native call, and the general way beside an fp16 bias)
def test_a_step_whose_backward_is_beyond_the_kernels(dtype):
    M = dpa_mod("mxfp4")
    m = (1 << 24) + 32
    bias = None if dtype == torch.bfloat16 else torch.zeros(8, device="cuda", dtype=torch.float16)
    x, w = torch.zeros((m, 8), device="cuda", dtype=dtype), torch.ones((8, 8), device="cuda", dtype=dtype)
    x[-1] = 1.0
    y = M.linear_mxfp4_fwd(x, w, bias)
    assert torch.equal(y[-1], torch.full((8,), 8.0, device="cuda", dtype=dtype)) and not y[:-1].any()
    with pytest.raises(ValueError, match="the product of dweight"):
        M.linear_mxfp4_train_fwd(x, w, bias)
    w.requires_grad_()
    with pytest.raises(ValueError, match="the product of dweight"):
        M.linear_mxfp4(x, w, bias)
    # without that gradient the step is taken
    w.requires_grad_(False)
    x.requires_grad_()
    y = M.linear_mxfp4(x, w, bias)
    y.backward(torch.ones((1, 1), device="cuda", dtype=dtype).expand_as(y))
    assert bool((x.grad == 8.0).all())
