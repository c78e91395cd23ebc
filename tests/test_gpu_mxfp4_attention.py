"""Cross attention over keys and values in MXFP4 against the definition in 64 bits.

Errors: a score's fp32 sum (D + 2 steps of 2^-23 of the magnitudes' sum) and two roundings of its factor move
its probability by that much relative to it; the exponential by 2^-21; the probability is rounded to the operands'
type for the product with the values (half a step), the output once more."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import mxfp4_reference as R
from conftest import dpa_mod

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    return dpa_mod("mxfp4")


def make(b, lq, lk, h, g, d, dtype, seed=1, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    q = (torch.randn((b, lq, h, d), generator=gen) * std).to(dtype)
    kv = torch.randn((b, lk, 2, g, d), generator=gen).to(dtype)
    return q, kv, M_quant(kv)


def M_quant(kv):
    """(codes, bytes, values in 64 bits) by the definition"""
    code, byte = R.quantize(kv)
    return code, byte, R.values_of(code, byte)


def packed(M, q4):
    code, byte, _ = q4
    return M.MXFP4(R.pack(code).cuda(), torch.from_numpy(byte.astype(np.uint8)).cuda())


def check(q, values, seen, out, lse, dtype, scale=None):
    """seen [b, lk] bool; rows of values that are not seen take no part"""
    b, lq, h, d = q.shape
    g = values.shape[3]
    scale = 1 / math.sqrt(d) if scale is None else scale
    half = torch.finfo(dtype).eps / 2
    out, lse = out.cpu().double(), lse.cpu().double()
    for i in range(b):
        at = seen[i].nonzero()[:, 0]
        if at.numel() == 0:
            assert (out[i] == 0).all() and (lse[i] == -math.inf).all()
            continue
        for j in range(h):
            k, v = values[i, at, 0, j * g // h], values[i, at, 1, j * g // h]
            x = q[i, :, j].double()
            s = scale * (x @ k.t())
            size = scale * (x.abs() @ k.abs().t())
            want_lse = torch.logsumexp(s, 1)
            p = torch.exp(s - want_lse[:, None])
            want = p @ v
            ds = ((d + 4) * 2.0**-23 * size).amax(1, keepdim=True) + 2.0**-23 * s.abs().amax(1, keepdim=True) + 2.0**-20
            pv = p @ v.abs()
            n = at.numel()
            bound = (2 * ds + half + (n + 2) * 2.0**-23) * pv + half * want.abs() + 2.0**-24
            err = (out[i, :, j] - want).abs()
            assert (err <= bound).all(), (i, j, float((err / bound).max()))
            el = (lse[i, j] - want_lse).abs()
            assert (el <= ds[:, 0] + n * 2.0**-23 + 2.0**-22 * want_lse.abs()).all(), (i, j, float(el.max()))


SIZES = [(1, 1, 1, 1, 1, 32), (2, 1, 77, 4, 4, 64), (3, 1, 300, 8, 2, 128), (2, 1, 2000, 16, 2, 96), (1, 7, 33, 2, 1, 32),
         (2, 40, 130, 4, 4, 64), (2, 256, 77, 4, 4, 32), (1, 1024, 64, 2, 2, 128), (2, 300, 500, 8, 4, 96),
         (64, 130, 65, 4, 4, 64), (40, 150, 129, 8, 8, 32), (32, 200, 100, 8, 8, 128), (1, 3, 9000, 4, 1, 64)]


@pytest.mark.parametrize("b,lq,lk,h,g,d", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mask", ["none", "lengths", "bool", "both"])
def test_attention(M, b, lq, lk, h, g, d, dtype, mask):
    print(f"attention {(b, lq, lk, h, g, d)} {dtype} {mask}", flush=True)
    q, _, q4 = make(b, lq, lk, h, g, d, dtype)
    code, byte, values = q4
    gen = torch.Generator().manual_seed(2)
    seen = torch.ones((b, lk), dtype=torch.bool)
    lengths = key_mask = None
    if mask in ("lengths", "both"):
        lengths = torch.randint(0, lk + 1, (b,), generator=gen)
        lengths[0] = lk
        if b > 1:
            lengths[1] = 0
        if b > 2:
            lengths[2] = 1
        seen &= torch.arange(lk) < lengths[:, None]
    if mask in ("bool", "both"):
        key_mask = torch.rand((b, lk), generator=gen) < 0.7
        key_mask[-1] = False
        seen &= key_mask
    # what takes no part holds nothing
    byte = byte.copy()
    byte[~seen.numpy()] = 255
    kv = packed(M, (code, byte, None))
    kw = dict(key_lengths=None if lengths is None else lengths.cuda(), key_mask=None if key_mask is None else key_mask.cuda())
    out, lse = M.cross_attention_mxfp4_fwd(q.cuda(), kv, **kw)
    assert out.dtype == dtype and lse.dtype == torch.float32
    check(q, values, seen, out, lse, dtype)
    again = M.cross_attention_mxfp4_fwd(q.cuda(), kv, **kw)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    assert torch.equal(M.cross_attention_mxfp4(q.cuda(), kv, **kw), out)


@pytest.mark.parametrize("lq", [1, 200])
def test_attention_agrees_with_the_cache_kept_whole(M, lq):
    """The same operator over the dequantised keys and values, which bf16 holds."""
    C = dpa_mod("conditioning")
    q, kv, _ = make(3, lq, 700, 8, 4, 64, torch.bfloat16)
    q4 = M.quantize_mxfp4(kv.cuda())
    full = M.dequantize_mxfp4(q4)
    out, lse = M.cross_attention_mxfp4_fwd(q.cuda(), q4)
    ref, ref_lse = C.cross_attention_fwd(q.cuda(), full[:, :, 0], full[:, :, 1])
    assert (out.float() - ref.float()).abs().max() <= 2.0**-7 * float(ref.float().abs().max())
    assert torch.allclose(lse, ref_lse, atol=1e-5, rtol=0)


@pytest.mark.parametrize("lq", [1, 150])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_attention_reads_views_in_place_and_copies_the_rest(M, lq, d):
    b, lk, h, g = 3, 90, 4, 2
    q, _, q4 = make(b, lq, lk, h, g, d, torch.bfloat16, seed=4)
    kv = packed(M, q4)
    seen = torch.ones((b, lk), dtype=torch.bool)
    out, lse = M.cross_attention_mxfp4_fwd(q.cuda(), kv)
    check(q, q4[2], seen, out, lse, torch.bfloat16)
    # a part of a longer cache, its other rows NaN
    long = M.MXFP4(torch.full((b, lk + 40, 2, g, d // 2), 0x77, dtype=torch.uint8, device="cuda"),
                   torch.full((b, lk + 40, 2, g, d // 32), 255, dtype=torch.uint8, device="cuda"))
    for part, src in zip(long, kv):
        part[:, 16:16 + lk] = src
    cut = M.MXFP4(*(t[:, 16:16 + lk] for t in long))
    assert torch.equal(M.cross_attention_mxfp4_fwd(q.cuda(), cut)[0], out)
    # one prompt for every image
    one = M.MXFP4(*(t[:1].expand(b, -1, -1, -1, -1) for t in kv))
    ref = M.cross_attention_mxfp4_fwd(q.cuda(), M.MXFP4(*(t.contiguous() for t in one)))[0]
    assert torch.equal(M.cross_attention_mxfp4_fwd(q.cuda(), one)[0], ref)
    # heads before tokens, a base that is not 16-B aligned, scales that are not dense
    turned = M.MXFP4(*(t.permute(0, 3, 2, 1, 4).contiguous().permute(0, 3, 2, 1, 4) for t in kv))
    assert torch.equal(M.cross_attention_mxfp4_fwd(q.cuda(), turned)[0], out)
    odd = torch.empty(kv.data.numel() + 8, dtype=torch.uint8, device="cuda")[8:].view(kv.data.shape)
    odd.copy_(kv.data)
    loose = torch.stack((kv.scales, kv.scales), -1)[..., 0]
    assert torch.equal(M.cross_attention_mxfp4_fwd(q.cuda(), M.MXFP4(odd, loose))[0], out)
    # queries with their heads outside
    qt = q.cuda().transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(M.cross_attention_mxfp4_fwd(qt, kv)[0], out)


def test_attention_scales_at_both_ends_and_nan_of_a_visible_key(M):
    """Blocks at the smallest and largest powers a bf16 tensor can have, and a key that is NaN."""
    b, lq, lk, h, d = 1, 40, 50, 2, 64
    q, kv, _ = make(b, lq, lk, h, h, d, torch.bfloat16, seed=6)
    kv[:, :, 0, :, 32:] *= 2.0**-120
    kv[:, :, 1, 0] *= 2.0**100
    kv[:, :, 1, 1] *= 2.0**-120
    for n in (1, lq):
        q4 = M_quant(kv)
        out, lse = M.cross_attention_mxfp4_fwd(q[:, :n].cuda(), packed(M, q4))
        for j, unit in ((0, 2.0**100), (1, 2.0**-120)):
            check(q[:, :n, j:j + 1], torch.cat((q4[2][:, :, :1, j:j + 1], q4[2][:, :, 1:, j:j + 1] / unit), 2),
                  torch.ones((b, lk), dtype=torch.bool), out[:, :, j:j + 1].cpu().double() / unit, lse[:, j:j + 1],
                  torch.bfloat16)
        bad = kv.clone()
        bad[0, 3, 0, 1, 5] = math.nan
        out, lse = M.cross_attention_mxfp4_fwd(q[:, :n].cuda(), packed(M, M_quant(bad)))
        assert torch.isnan(out[:, :, 1]).all() and torch.isfinite(out[:, :, 0]).all()
        bad = kv.clone()
        bad[0, 3, 1, 1, 5] = math.inf
        out, lse = M.cross_attention_mxfp4_fwd(q[:, :n].cuda(), packed(M, M_quant(bad)))
        assert torch.isnan(out[:, :, 1, :32]).all() and torch.isfinite(out[:, :, 1, 32:]).all()


def test_attention_without_keys_or_queries(M):
    q, _, q4 = make(2, 5, 8, 2, 2, 64, torch.bfloat16)
    kv = packed(M, q4)
    none = M.MXFP4(*(t[:, :0] for t in kv))
    out, lse = M.cross_attention_mxfp4_fwd(q.cuda(), none)
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = M.cross_attention_mxfp4_fwd(q[:, :0].cuda(), kv)
    assert out.shape == (2, 0, 2, 64) and lse.shape == (2, 2, 0)


def test_attention_in_a_graph_and_on_another_stream(M):
    q, _, q4 = make(4, 1, 5000, 8, 2, 128, torch.bfloat16)
    kv, qs = packed(M, q4), q.cuda()
    lengths = torch.tensor([5000, 17, 0, 4097], dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        M.cross_attention_mxfp4_fwd(qs, kv, key_lengths=lengths)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = M.cross_attention_mxfp4_fwd(qs, kv, key_lengths=lengths)
    for i in range(4):
        lengths.copy_(torch.tensor([5000 - i, 17 + i, i, 4097]))
        qs.mul_(0.9)
        graph.replay()
        want = M.cross_attention_mxfp4_fwd(qs, kv, key_lengths=lengths)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
