"""Attention over 4-bit keys and values in every form of its kernels and every head dim that each has, against 64 bits on
the GPU. The bounds are those of test_gpu_mxfp4_attention.py: a score's fp32 sum and two roundings of its factor, the
exponential, the probability in the operands' type, the output's half step."""
from __future__ import annotations

import math

import pytest
import torch

from conftest import dpa_mod

pytestmark = pytest.mark.gpu

# (batch, queries, keys, query heads, key heads, head dim); rows: queries of all query heads of a key head
MANY = [(20, 150, 200, 8, 8, 64), (20, 150, 200, 8, 8, 96), (20, 150, 200, 8, 8, 128), (40, 70, 333, 8, 4, 64), (40, 33, 1031, 8, 8, 128),
        (16, 260, 700, 4, 2, 32), (16, 260, 1100, 4, 2, 64), (16, 260, 1100, 4, 2, 96), (16, 260, 1100, 4, 2, 128)]     # (1100: split)
FEW = [(2, 17, 300, 4, 4, 32), (3, 20, 1500, 4, 2, 32), (1, 32, 5000, 8, 8, 64), (2, 25, 2100, 4, 4, 96), (2, 17, 300, 4, 4, 128),
       (3, 20, 1500, 4, 2, 128), (2, 100, 200, 2, 2, 128)]
TOKEN = [(5, 2, 4097, 8, 2, 64), (3, 1, 2500, 4, 4, 32), (2, 3, 1200, 10, 2, 96), (3, 16, 129, 4, 4, 128)]


def test_the_sizes_take_their_forms():
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    for sizes, form in ((MANY, "many"), (FEW, "few"), (TOKEN, "token")):
        for b, lq, lk, h, g, _ in sizes:
            rows = lq * h // g
            assert lk > 128
            few = rows <= 32 or b * g * -(-rows // 32) < 2 * cus
            assert form == ("token" if rows <= 16 else "few" if few else "many"), (b, lq, lk, h, g)


def check(q, values, seen, out, lse):
    dtype, (b, lq, h, d), g = q.dtype, q.shape, values.shape[3]
    half, r = torch.finfo(dtype).eps / 2, h // g
    out, lse = out.double(), lse.double()
    for i in range(b):
        at = seen[i].nonzero()[:, 0]
        n = at.numel()
        if n == 0:
            assert not out[i].any() and (lse[i] == -math.inf).all()
            continue
        x = q[i].double().view(lq, g, r, d).permute(1, 2, 0, 3).reshape(g, r * lq, d)
        k, v = (values[i, at, j].transpose(0, 1).contiguous() for j in (0, 1))     # [g, n, d]
        kt = k.transpose(1, 2).contiguous()
        s = torch.matmul(x, kt) / math.sqrt(d)
        size = torch.matmul(x.abs(), kt.abs()) / math.sqrt(d)
        want_lse = torch.logsumexp(s, 2)
        p = torch.exp(s - want_lse[..., None])
        want, pv = torch.matmul(p, v), torch.matmul(p, v.abs())
        ds = ((d + 4) * 2.0**-23 * size).amax(2, keepdim=True) + 2.0**-23 * s.abs().amax(2, keepdim=True) + 2.0**-20
        got = out[i].view(lq, g, r, d).permute(1, 2, 0, 3).reshape(g, r * lq, d)
        bound = (2 * ds + half + (n + 2) * 2.0**-23) * pv + half * want.abs() + 2.0**-24
        assert ((got - want).abs() <= bound).all(), (i, float(((got - want).abs() / bound).max()))
        el = (lse[i].reshape(g, r * lq) - want_lse).abs()
        assert (el <= ds[..., 0] + n * 2.0**-23 + 2.0**-22 * want_lse.abs()).all(), (i, float(el.max()))


@pytest.mark.parametrize("size", MANY + FEW + TOKEN)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mask", ["none", "lengths", "bool", "both"])
def test_attention(size, dtype, mask):
    M = dpa_mod("mxfp4")
    print(f"attention {size} {dtype} {mask}", flush=True)
    b, lq, lk, h, g, d = size
    gen = torch.Generator("cuda").manual_seed(lq + lk + d)
    q = torch.randn((b, lq, h, d), generator=gen, device="cuda").to(dtype)
    kv = M.quantize_mxfp4(torch.randn((b, lk, 2, g, d), generator=gen, device="cuda").to(dtype))
    values = M.dequantize_mxfp4(kv, torch.float32).double()
    seen = torch.ones((b, lk), dtype=torch.bool, device="cuda")
    lengths = key_mask = None
    if mask in ("lengths", "both"):
        lengths = torch.randint(0, lk + 1, (b,), generator=gen, device="cuda")
        lengths[0] = lk
        if b > 1:
            lengths[1] = 0
        if b > 2:
            lengths[2] = 1
        seen &= torch.arange(lk, device="cuda") < lengths[:, None]
    if mask in ("bool", "both"):
        key_mask = torch.rand((b, lk), generator=gen, device="cuda") < 0.7
        key_mask[-1] = False
        seen &= key_mask
    kv.scales[~seen] = 255      # what takes no part holds nothing
    out, lse = M.cross_attention_mxfp4_fwd(q, kv, key_lengths=lengths, key_mask=key_mask)
    check(q, values, seen, out, lse)
    again = M.cross_attention_mxfp4_fwd(q, kv, key_lengths=lengths, key_mask=key_mask)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
