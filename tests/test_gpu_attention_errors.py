"""Cross attention's outputs and gradients against 64 bits as wholes (``attention_errors``: a tensor's and
each head's error against the roundings' expected one), where the elementwise bounds of
test_gpu_conditioning.py are too wide to show a fault: over long key axes, and in fp16."""
from __future__ import annotations

import math

import pytest
import torch

import attention_errors as E
from conftest import dpa_mod

pytestmark = pytest.mark.gpu

C = dpa_mod("conditioning")

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _mask(b, lk, kind, seed):
    g = torch.Generator().manual_seed(seed)
    lengths = mask = None
    seen = torch.ones((b, lk), dtype=torch.bool)
    if kind in ("lengths", "both"):
        lengths = torch.randint(lk // 2, lk + 1, (b,), generator=g).int()
        lengths[-1] = 0 if b > 1 else lk
        seen &= torch.arange(lk) < lengths[:, None]
    if kind in ("bool", "both"):
        mask = torch.rand((b, lk), generator=g) < 0.8
        if lk > 200:
            mask[0, 64:128] = False
        seen &= mask
    return lengths, mask, seen


def _run(dtype, b, lq, lk, h, kvh, d, kind, **kw):
    q, kv, dout = E.inputs(DT[dtype], b, lq, lk, h, kvh, d, seed=7 * lq + lk, **kw)
    lengths, mask, seen = _mask(b, lk, kind, lq + lk)
    kv[~seen] = float("nan")
    q, kv, dout, seen = (t.cuda() for t in (q, kv, dout, seen))
    masks = dict(key_lengths=None if lengths is None else lengths.cuda(),
                 key_mask=None if mask is None else mask.cuda())
    k, v = kv[:, :, 0], kv[:, :, 1]
    out, lse = C.cross_attention_fwd(q, k, v, **masks)
    dq, dk, dv = C.cross_attention_bwd(dout, q, k, v, out, lse, **masks)
    torch.cuda.synchronize()
    ref = E.reference(q, k, v, dout, seen, 1.0 / math.sqrt(d))
    for name in ("out", "dq", "dk", "dv"):
        assert float(ref[name][0].abs().max()) < (65504 if dtype == "fp16" else 1e38), name
    E.check(dict(out=out, dq=dq, dk=dk, dv=dv), ref)


FORMS = [
    # up to 128 keys; few rows; rows and keys in tiles; keys and rows split
    ("bf16", 3, 256, 77, 4, 4, 64, "lengths"),
    ("fp16", 3, 256, 77, 4, 4, 64, "bool"),
    ("fp16", 4, 300, 120, 4, 2, 32, "both"),
    ("bf16", 2, 700, 128, 2, 1, 128, "none"),
    ("bf16", 2, 1, 4500, 4, 1, 128, "lengths"),
    ("fp16", 2, 1, 4500, 8, 2, 64, "bool"),
    ("fp16", 1, 3, 2049, 8, 8, 64, "none"),
    ("bf16", 2, 1, 17000, 1, 1, 32, "bool"),
    ("bf16", 1, 50, 17000, 1, 1, 8, "none"),
    ("fp16", 1, 70, 9000, 2, 2, 64, "none"),
    ("fp16", 2, 300, 700, 2, 1, 96, "both"),
    ("bf16", 2, 1100, 1031, 4, 2, 64, "bool"),
    ("fp16", 6, 1000, 320, 8, 2, 64, "lengths"),
    ("bf16", 3, 600, 900, 4, 4, 128, "none"),
    ("fp16", 40, 300, 200, 4, 4, 64, "both"),
]


@pytest.mark.parametrize("offset", [0.0, 1.0])
@pytest.mark.parametrize("shape", FORMS)
def test_errors_are_the_roundings(shape, offset):
    print(f"attention {shape} offset={offset}", flush=True)
    _run(*shape, offset=offset)


FP16 = [
    ("fp16", 4, 256, 77, 4, 4, 64, "lengths"),
    ("fp16", 2, 300, 128, 2, 1, 128, "none"),
    ("fp16", 3, 1500, 50, 2, 2, 32, "bool"),
    ("fp16", 2, 1, 4500, 4, 1, 128, "none"),
    ("fp16", 1, 3, 2049, 8, 8, 64, "bool"),
    ("fp16", 1, 1100, 4096, 2, 2, 64, "none"),
    ("fp16", 2, 300, 700, 2, 1, 96, "both"),
    ("fp16", 6, 1000, 192, 8, 2, 64, "lengths"),
    ("fp16", 40, 300, 200, 4, 4, 32, "none"),
]


@pytest.mark.parametrize("std", [1e-5, 1e-4, 1e-2, 300.0])
@pytest.mark.parametrize("shape", FP16)
def test_fp16_gradients_of_any_size(shape, std):
    """Gradients as they come without a loss scale and with a large one."""
    print(f"attention {shape} dout std={std}", flush=True)
    _run(*shape, dout_std=std)


@pytest.mark.parametrize("lk", [40, 120, 900])
def test_fp16_gradients_that_grow_along_an_axis(lk):
    """Rows, and values, whose magnitudes span 2^16 in either order: what a kernel stands at has to follow."""
    for order in (1, -1):
        for axis in ("rows", "keys"):
            q, kv, dout = E.inputs(torch.float16, 2, 500, lk, 2, 2, 64, seed=lk)
            ramp = torch.exp2(torch.linspace(-10, 6, 500 if axis == "rows" else lk))
            ramp = ramp.flip(0) if order < 0 else ramp
            if axis == "rows":
                dout = (dout.float() * ramp[:, None, None]).half()
            else:
                kv[:, :, 1] = (kv[:, :, 1].float() * ramp[:, None, None]).half()
            print(f"lk={lk} order={order} axis={axis}", flush=True)
            q, kv, dout = q.cuda(), kv.cuda(), dout.cuda()
            k, v = kv[:, :, 0], kv[:, :, 1]
            out, lse = C.cross_attention_fwd(q, k, v)
            dq, dk, dv = C.cross_attention_bwd(dout, q, k, v, out, lse)
            seen = torch.ones((2, lk), dtype=torch.bool, device="cuda")
            E.check(dict(out=out, dq=dq, dk=dk, dv=dv), E.reference(q, k, v, dout, seen, 0.125))


def test_fp16_gradients_that_are_zero_or_not_finite():
    """Zero gradients give zeros; an infinite or NaN one reaches its own head's gradients alone."""
    for lq, lk in ((1, 300), (200, 77), (200, 300)):
        q, kv, _ = (t.cuda() for t in E.inputs(torch.float16, 2, lq, lk, 2, 2, 64, seed=3))
        k, v = kv[:, :, 0], kv[:, :, 1]
        out, lse = C.cross_attention_fwd(q, k, v)
        zero = torch.zeros_like(q)
        assert not any(t.any() for t in C.cross_attention_bwd(zero, q, k, v, out, lse))
        one = torch.randn(q.shape, generator=torch.Generator().manual_seed(4)).half().cuda()
        want = C.cross_attention_bwd(one, q, k, v, out, lse)
        for bad in (float("inf"), float("nan")):
            dout = one.clone()
            dout[0, 0, 1, 5] = bad
            got = C.cross_attention_bwd(dout, q, k, v, out, lse)
            assert not got[0][0, 0, 1].isfinite().all() and not got[2][0, :, 1].isfinite().all()
            for a, w in zip(got, want):
                assert torch.equal(a[1], w[1]) and torch.equal(a[0, :, 0], w[0, :, 0])
