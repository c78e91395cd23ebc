"""The MXFP4 product in every form of its kernel, whole outputs against 64 bits: sums of K + 2 fp32 steps, each within a
step of the sum of magnitudes, and the output's half step."""
from __future__ import annotations

import math

import pytest
import torch

from conftest import dpa_mod
from mxfp4_forms import DTYPES, FORMS, check_plan

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    return dpa_mod("mxfp4")


def rounded(M, x):
    """x as its operand holds it, in 64 bits (quantisation and back are exact, blocks of a row's end filled with zeros)"""
    k = x.shape[1]
    whole = torch.nn.functional.pad(x, (0, -k % 32))
    return M.dequantize_mxfp4(M.quantize_mxfp4(whole), torch.float32)[:, :k].double().contiguous()


@pytest.mark.parametrize("size", FORMS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_product(M, size, dtype):
    m, n, k = size
    print(f"product {size} {dtype}", flush=True)
    check_plan(size, dtype)
    g = torch.Generator("cuda").manual_seed(m + n + k)
    x = torch.randn((m, k), generator=g, device="cuda").to(dtype)
    w = (torch.randn((n, k), generator=g, device="cuda") / math.sqrt(k)).to(dtype)
    bias = torch.randn(n, generator=g, device="cuda") if m % 8 else None
    kept = M.mxfp4_operand(w)
    y = M.linear_mxfp4_fwd(x, kept, bias)
    again = M.linear_mxfp4_fwd(x, kept, bias)
    assert torch.equal(y, again)
    a, b = rounded(M, x), rounded(M, w).t().contiguous()
    want, size_of_sums = a @ b, a.abs() @ b.abs()
    if bias is not None:
        want += bias.double()
        size_of_sums += bias.double().abs()
    sums = (k + 2) * 2.0**-23 * size_of_sums
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    over = (y.double() - want).abs() - (sums + torch.finfo(dtype).eps / 2 * (want.abs() + sums) + tiny)
    assert float(over.max()) <= 0, divmod(int(over.argmax()), n)
