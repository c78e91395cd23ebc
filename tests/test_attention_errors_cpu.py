"""The comparison of ``attention_errors`` passes what only rounds, and rejects small faults over long
key axes."""
from __future__ import annotations

import math

import pytest
import torch

import attention_errors as E

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
SHAPES = [
    ("bf16", 1, 1, 1, 1, 1, 64), ("bf16", 5, 1, 77, 4, 4, 64), ("fp16", 3, 1, 130, 4, 2, 64),
    ("bf16", 3, 33, 65, 2, 2, 128), ("fp16", 2, 129, 200, 3, 3, 80), ("bf16", 2, 1, 4500, 4, 1, 128),
    ("fp16", 1, 3, 2049, 8, 8, 64), ("bf16", 2, 1, 17000, 1, 1, 32), ("bf16", 1, 50, 17000, 1, 1, 8),
    ("fp16", 1, 300, 700, 2, 1, 96),
]
LONG = [s for s in SHAPES if s[3] >= 2000]


def _case(dtype, b, lq, lk, h, kvh, d, **kw):
    q, kv, dout = E.inputs(DT[dtype], b, lq, lk, h, kvh, d, seed=lq + lk, **kw)
    seen = torch.ones((b, lk), dtype=torch.bool)
    if b > 1:
        seen[1, lk // 2:] = False
    if b > 2:
        seen[2] = False
    return q, kv[:, :, 0], kv[:, :, 1], dout, seen, 1.0 / math.sqrt(d)


@pytest.mark.parametrize("offset", [0.0, 1.0])
@pytest.mark.parametrize("shape", SHAPES)
def test_roundings_pass(shape, offset):
    args = _case(*shape, offset=offset)
    E.check(E.simulate(*args), E.reference(*args))


@pytest.mark.parametrize("shape", LONG)
def test_faults_are_rejected(shape):
    args = _case(*shape, offset=1.0)
    ref = E.reference(*args)

    def over(got, *names):
        e = E.excess(got, ref)
        return all(max(e[n]) > 1 for n in names)
    assert over(E.simulate(*args, drop=128), "out", "dq")
    assert over(E.simulate(*args, no_d=True), "dq", "dk")
    right = E.simulate(*args)
    for name in ("out", "dq", "dk", "dv"):
        assert over({name: torch.zeros_like(right[name])}, name)
    plain = _case(*shape)
    e = E.excess(E.simulate(*plain, drop=128), E.reference(*plain))
    assert max(e["out"]) > 1 and max(e["dq"]) > 1


@pytest.mark.parametrize("std", [1e-4, 1e-5])
def test_fp16_gradients_below_its_range_are_rejected(std):
    """dS of small gradients over many keys, rounded to fp16 as it is, loses most of its bits; scaled it
    does not."""
    args = _case("fp16", 1, 64, 4096, 2, 2, 64, dout_std=std)
    ref = E.reference(*args)
    E.check(E.simulate(*args), ref)
    e = E.excess(E.simulate(*args, scaled=False), ref)
    assert max(e["dq"]) > 1
