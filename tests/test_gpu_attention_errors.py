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
