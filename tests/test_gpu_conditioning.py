"""The conditioning operators (cross attention, dropout, token embedding) against plain
implementations in 64 bits on the same inputs.

Tolerances are elementwise and count roundings. u = half a step of the operands' type relative to
the value (finfo.eps / 2: bf16 2^-8, fp16 2^-11). Cross attention: a probability p is off by
rel = 2^-19 + 2 (D + 8) 2^-24 max sum scale |q k| + 2^-21 (max |score| + |lse|), the fp32 products,
the exponent's argument and the exponential, and by u p (+ 2^-25 absolutely in fp16, whose
subnormals end there) where it is rounded for the product with v; outputs are rounded once more:
  |out - exact| <= (u + rel) sum p |v| + u |exact|  (sums over a row's keys)
The gradients follow from the same counts through D = rowsum(dout out), with out as rounded:
  |dD| <= sum |dout| |out - exact|,  |dds| <= p |dD| + (u + 2 rel) p (|dp| + |D|)
  |dq - exact| <= scale sum |dds| |k| + u |exact|, dk alike over queries, dv like out over queries.
fp32 sums of n terms add 2^-24 n of the terms' magnitudes. Dropout and the embedding's forward are
exact to the bit; the embedding's gradient adds n 2^-24 of the summed magnitudes and one rounding.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from conftest import dpa_mod

pytestmark = pytest.mark.gpu

C = dpa_mod("conditioning")

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- cross attention -----------------------------------------------------------------------
def _visible(b, lk, kind, g):
    """(key_lengths, key_mask, visible [b, lk])"""
    lengths = mask = None
    seen = torch.ones((b, lk), dtype=torch.bool)
    if kind in ("lengths", "both"):
        lengths = torch.randint(0, lk + 1, (b,), generator=g)
        lengths[0] = lk
        if b > 1:
            lengths[1] = 0
        if b > 2:
            lengths[2] = lk + 7           # clamped
        if b > 3:
            lengths[3] = -3
        lengths = lengths.to(torch.int32)
        seen &= torch.arange(lk) < lengths[:, None]
    if kind in ("bool", "both"):
        mask = torch.rand((b, lk), generator=g) < 0.7
        if b > 1:
            mask[1] = False
        if lk > 130:
            mask[0, 64:128] = False       # a whole tile
        seen &= mask
    return lengths, mask, seen


def _case(dtype, b, lq, lk, h, kvh, d, kind, seed=0, std=1.0):
    g = _gen(seed)
    dt = DT[dtype]
    q = (torch.randn((b, lq, h, d), generator=g) * std).to(dt)
    kv = (torch.randn((b, lk, 2, kvh, d), generator=g) * std).to(dt)
    dout = torch.randn((b, lq, h, d), generator=g).to(dt)
    lengths, mask, seen = _visible(b, lk, kind, g)
    kv[~seen] = float("nan")              # never read
    dev = [None if t is None else t.cuda() for t in (q, kv, dout, lengths, mask)]
    return (*dev, seen)


def _reference(q, k, v, dout, seen, scale):
    """Formula and tolerances in 64 bits: {name: (exact, bound)}."""
    u = HALF[q.dtype]
    sub = 2.0**-25 if q.dtype == torch.float16 else 0.0
    b, lq, h, d = q.shape
    lk, kvh = k.shape[1:3]
    rep = h // kvh

    def heads(t, n=1):
        return t.double().transpose(1, 2).repeat_interleave(n, 1)
    vis = seen.to(q.device)[:, None, None, :]
    q_, do = heads(q), heads(dout)
    k_, v_ = (torch.where(vis.transpose(2, 3), heads(t, rep), 0.0) for t in (k, v))
    x = (q_ @ k_.transpose(2, 3)) * scale
    mag = (q_.abs() @ k_.abs().transpose(2, 3)) * scale
    x = torch.where(vis, x, -math.inf)
    top = x.amax(3, keepdim=True) if lk else torch.full((b, h, lq, 1), -math.inf, device=q.device).double()
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(x - top)
    tot = e.sum(3, keepdim=True)
    p = e / torch.where(tot == 0, 1.0, tot)
    lse = (top + torch.log(tot)).squeeze(3)
    o = p @ v_
    fin = torch.where(vis, x.abs(), 0.0)
    big = fin.amax(3, keepdim=True) if lk else torch.zeros_like(top)
    rel = (2.0**-19 + 2 * (d + 8) * 2.0**-24 * (mag.amax(3, keepdim=True) if lk else 0.0)
           + 2.0**-21 * (big + torch.where(lse.isfinite(), lse.abs(), 0.0)[..., None])
           + lk * 2.0**-24)
    pv = torch.where(vis, p, 0.0)
    b_o = (u + rel) * (pv @ v_.abs()) + sub * (vis * v_.abs().transpose(2, 3).sum(2, keepdim=True)).sum(3, keepdim=True) / max(1, d) * d + u * o.abs() if lk else torch.zeros_like(o)
    dp = do @ v_.transpose(2, 3)
    dpm = do.abs() @ v_.abs().transpose(2, 3)
    dd = (do * o).sum(3, keepdim=True)
    ds = p * (dp - dd)
    b_dd = (do.abs() * b_o).sum(3, keepdim=True) + d * 2.0**-24 * (do * o).abs().sum(3, keepdim=True)
    b_ds = pv * b_dd + (u + 2 * rel) * pv * (dp.abs() + dd.abs()) + pv * (d + 2) * 2.0**-24 * dpm + sub
    b_ds = torch.where(vis, b_ds, 0.0)
    rows = lq * rep * 2.0**-24
    dq, b_dq = scale * (ds @ k_), scale * ((b_ds + lk * 2.0**-24 * ds.abs()) @ k_.abs())
    dk, b_dk = scale * (ds.transpose(2, 3) @ q_), scale * ((b_ds + rows * ds.abs()).transpose(2, 3) @ q_.abs())
    dv = p.transpose(2, 3) @ do
    b_dv = ((pv * (u + rel + rows)) + torch.where(vis, sub, 0.0)).transpose(2, 3) @ do.abs()

    def out(t):
        return t.transpose(1, 2)

    def shared(t):
        return t.view(b, kvh, rep, lk, d).sum(2).transpose(1, 2)
    res = {"out": (out(o), out(b_o)), "dq": (out(dq), out(b_dq + u * dq.abs()))}
    res["dk"] = (shared(dk), shared(b_dk))
    res["dv"] = (shared(dv), shared(b_dv))
    for n in ("dk", "dv"):
        res[n] = (res[n][0], res[n][1] + u * res[n][0].abs())
    b_lse = torch.where(lse.isfinite(), rel.squeeze(3) + 2.0**-22 * lse.abs(), 0.0)
    res["lse"] = (lse, b_lse)
    # numbers below the type's normal range round to its subnormal steps
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    return {n: (a, bound + (tiny if n != "lse" else 0.0)) for n, (a, bound) in res.items()}


def _compare(got, ref):
    for name, t in got.items():
        exact, bound = ref[name]
        assert t.shape == exact.shape, name
        t = t.double()
        inf = exact.isinf()
        assert torch.equal(t[inf], exact[inf]), name
        diff = torch.where(inf, 0.0, (t - exact).abs())
        over = diff - torch.where(inf, 0.0, bound)
        worst = float(over.max()) if over.numel() else 0.0
        assert worst <= 0 and bool(diff.isfinite().all()), (
            f"{name}: {int((over > 0).sum())} of {over.numel()} beyond the bound, worst by {worst:.3e}")


SHAPES = [
    # dtype, batch, lq, lk, heads, kv heads, dim, mask
    ("bf16", 1, 1, 1, 1, 1, 8, "none"),
    ("bf16", 5, 1, 77, 4, 4, 64, "lengths"),
    ("fp16", 3, 1, 130, 4, 2, 64, "bool"),
    ("bf16", 2, 7, 33, 4, 1, 40, "bool"),
    ("fp16", 4, 32, 64, 2, 2, 32, "lengths"),
    ("bf16", 3, 33, 65, 2, 2, 128, "both"),
    ("fp16", 2, 16, 31, 6, 3, 24, "none"),
    ("fp16", 2, 129, 200, 3, 3, 80, "bool"),
    ("bf16", 4, 256, 77, 4, 4, 64, "lengths"),
    ("bf16", 5, 100, 77, 4, 4, 32, "lengths"),
    ("fp16", 1, 300, 700, 2, 1, 96, "none"),
    ("bf16", 2, 64, 1031, 8, 2, 128, "both"),
    ("bf16", 2, 1, 4500, 4, 1, 128, "lengths"),
    ("fp16", 1, 3, 2049, 8, 8, 64, "bool"),
    ("bf16", 1, 1100, 513, 2, 2, 64, "bool"),
    ("fp16", 1, 2050, 40, 1, 1, 72, "none"),
    ("bf16", 2, 1, 17000, 1, 1, 32, "bool"),       # more keys than one workgroup's range
    ("bf16", 1, 50, 17000, 1, 1, 8, "lengths"),
]


@pytest.mark.parametrize("dtype,b,lq,lk,h,kvh,d,kind", SHAPES)
def test_attention_against_64_bits(dtype, b, lq, lk, h, kvh, d, kind):
    print(f"attention {dtype} b={b} lq={lq} lk={lk} h={h}/{kvh} d={d} {kind}", flush=True)
    q, kv, dout, lengths, mask, seen = _case(dtype, b, lq, lk, h, kvh, d, kind, seed=lq + lk)
    k, v = kv[:, :, 0], kv[:, :, 1]
    scale = 1.0 / math.sqrt(d)
    kw = dict(key_lengths=lengths, key_mask=mask)
    out, lse = C.cross_attention_fwd(q, k, v, **kw)
    torch.cuda.synchronize()
    print("forward done", flush=True)
    dq, dk, dv = C.cross_attention_bwd(dout, q, k, v, out, lse, **kw)
    torch.cuda.synchronize()
    ref = _reference(q, k, v, dout, seen, scale)
    _compare(dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv), ref)
    hidden = ~seen.cuda()
    assert not dk[hidden].any() and not dv[hidden].any()
    # the same bits again
    out2, lse2 = C.cross_attention_fwd(q, k, v, **kw)
    again = C.cross_attention_bwd(dout, q, k, v, out, lse, **kw)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    assert all(torch.equal(x, y) for x, y in zip((dq, dk, dv), again))


MORE = [
    # up to 128 keys: blocks of 32 that are empty, one tile and several, splits of the rows, every
    # padded head size
    ("bf16", 2, 130, 1, 2, 2, 64, "none"),
    ("fp16", 3, 128, 32, 2, 1, 32, "bool"),
    ("bf16", 5, 400, 33, 2, 2, 64, "lengths"),
    ("bf16", 1, 1500, 77, 2, 1, 40, "bool"),
    ("fp16", 5, 50, 96, 3, 3, 128, "both"),
    ("bf16", 4, 140, 97, 2, 2, 64, "lengths"),
    ("fp16", 4, 200, 128, 4, 2, 32, "both"),
    ("bf16", 5, 90, 97, 2, 2, 128, "bool"),
    ("bf16", 5, 600, 128, 1, 1, 24, "lengths"),
    # more: tiles at the length's border, whole tiles hidden, rows in both forms, heads that share keys
    # in tiles that lie in one head or in two
    ("bf16", 3, 64, 129, 2, 2, 64, "bool"),
    ("fp16", 6, 1000, 192, 8, 2, 64, "both"),
    ("bf16", 6, 1000, 320, 8, 2, 32, "lengths"),
    ("bf16", 40, 300, 200, 4, 4, 64, "both"),
    ("fp16", 20, 130, 640, 6, 3, 128, "lengths"),
    ("bf16", 9, 512, 1024, 8, 8, 64, "none"),
]


@pytest.mark.parametrize("dtype,b,lq,lk,h,kvh,d,kind", MORE)
def test_attention_forms_against_64_bits(dtype, b, lq, lk, h, kvh, d, kind):
    test_attention_against_64_bits(dtype, b, lq, lk, h, kvh, d, kind)
    # a frozen encoder: dq alone, the same bits
    q, kv, dout, lengths, mask, _ = _case(dtype, b, lq, lk, h, kvh, d, kind, seed=lq + lk)
    k, v = kv[:, :, 0], kv[:, :, 1]
    kw = dict(key_lengths=lengths, key_mask=mask)
    out, lse = C.cross_attention_fwd(q, k, v, **kw)
    both = C.cross_attention_bwd(dout, q, k, v, out, lse, **kw)
    alone = C._attention_bwd(dout, q, k, v, out, lse, lengths, mask, None, None, None)
    assert alone[1] is None and alone[2] is None and torch.equal(alone[0], both[0])


@pytest.mark.parametrize("lk", [50, 700])
def test_attention_far_strides(lk):
    """Rows of keys more than 2^24 elements apart and a whole cache past 2^31 of them."""
    step = (1 << 32) // lk // 8 * 8 if lk == 50 else (1 << 23) + 8
    room = torch.empty((lk - 1) * step + 2 * 64, device="cuda", dtype=torch.bfloat16)
    far = room.as_strided((1, lk, 2, 64), (0, step, 64, 1))
    g = _gen(41)
    q = torch.randn((1, 100, 4, 64), generator=g).bfloat16().cuda()
    near = torch.randn((1, lk, 2, 64), generator=g).bfloat16().cuda()
    far.copy_(near)
    a, c = C.cross_attention_fwd(q, far, far), C.cross_attention_fwd(q, near, near)
    assert all(torch.equal(x, y) for x, y in zip(a, c))
    dout = torch.randn(q.shape, generator=g).bfloat16().cuda()
    a = C.cross_attention_bwd(dout, q, far, far, *a)
    c = C.cross_attention_bwd(dout, q, near, near, *c)
    assert all(torch.equal(x, y) for x, y in zip(a, c))
    one = q[:, :1]
    a, c = C.cross_attention_fwd(one, far, far), C.cross_attention_fwd(one, near, near)
    assert all(torch.equal(x, y) for x, y in zip(a, c))


def test_attention_no_keys_many_queries():
    """Rows that would be split over workgroups, and no key to sum for."""
    q = torch.randn((1, 3000, 1, 64), device="cuda").bfloat16()
    k = q[:, :0]
    out, lse = C.cross_attention_fwd(q, k, k)
    dq, dk, dv = C.cross_attention_bwd(q, q, k, k, out, lse)
    assert not out.any() and bool((lse == -math.inf).all()) and not dq.any()
    assert dk.shape == (1, 0, 1, 64) and dv.shape == dk.shape


def test_attention_extreme_masked_scores():
    """Hidden keys whose scores would be the largest, rows whose scores are far below zero, and
    batches whose mask hides everything, in every form."""
    for lq, lk in ((1, 40), (70, 77), (70, 300), (300, 900)):
        q, kv, dout, _, _, _ = _case("bf16", 3, lq, lk, 2, 2, 64, "none", seed=51)
        mask = (torch.rand((3, lk), generator=_gen(52)) < 0.5).cuda()
        mask[2] = False
        kv = torch.where(mask[:, :, None, None, None], kv, torch.full_like(kv, 3e4))
        q = q.clone()
        q[0] *= 40.0                                   # scores of hundreds
        k, v = kv[:, :, 0], kv[:, :, 1]
        out, lse = C.cross_attention_fwd(q, k, v, key_mask=mask)
        grads = C.cross_attention_bwd(dout, q, k, v, out, lse, key_mask=mask)
        assert not out[2].any() and bool((lse[2] == -math.inf).all())
        assert all(t.isfinite().all() for t in (out, *grads))
        assert not grads[0][2].any() and not grads[1][2].any() and not grads[2][2].any()
        clean = torch.where(mask[:, :, None, None, None], kv, torch.zeros_like(kv))
        again = C.cross_attention_fwd(q, clean[:, :, 0], clean[:, :, 1], key_mask=mask)
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("lq,lk", [(0, 5), (3, 0), (0, 0), (40, 0)])
def test_attention_empty(lq, lk):
    q = torch.randn((2, lq, 4, 64), device="cuda").bfloat16()
    k = torch.randn((2, lk, 2, 64), device="cuda").bfloat16()
    out, lse = C.cross_attention_fwd(q, k, k)
    assert out.shape == q.shape and not out.any() and bool((lse == -math.inf).all())
    dq, dk, dv = C.cross_attention_bwd(torch.ones_like(q), q, k, k, out, lse)
    assert dq.shape == q.shape and dk.shape == k.shape and not dq.any() and not dk.any() and not dv.any()
    out, lse = C.cross_attention_fwd(q[:0], k[:0], k[:0])
    assert out.shape == (0, lq, 4, 64)
    assert [t.shape[0] for t in C.cross_attention_bwd(out, q[:0], k[:0], k[:0], out, lse)] == [0, 0, 0]


def test_attention_peaked_and_scaled():
    """Scores of hundreds, where all but one probability vanish, and a scale of the caller's."""
    for scale in (1.0, 0.02):
        q, kv, dout, _, _, seen = _case("bf16", 2, 70, 150, 2, 2, 64, "none", seed=5, std=4.0)
        k, v = kv[:, :, 0], kv[:, :, 1]
        out, lse = C.cross_attention_fwd(q, k, v, scale=scale)
        grads = C.cross_attention_bwd(dout, q, k, v, out, lse, scale=scale)
        _compare(dict(zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads))),
                 _reference(q, k, v, dout, seen, scale))


@pytest.mark.parametrize("lq", [3, 150])
def test_attention_strides(lq):
    """Operands that are not dense give what their dense copies give."""
    g = _gen(3)
    b, lk, h, kvh, d = 3, 90, 4, 2, 64
    q = torch.randn((b, h, lq, d), generator=g).bfloat16().cuda().transpose(1, 2)
    kv = torch.randn((b, lk, 2, kvh, d), generator=g).bfloat16().cuda()
    dout = torch.randn((lq, b, h, d), generator=g).bfloat16().cuda().transpose(0, 1)
    mask = (torch.rand((b, 2, lk), generator=g) < 0.8).cuda()[:, 1]
    lengths = torch.tensor([90, 17, 0], device="cuda")            # int64
    k, v = kv[:, :, 0], kv[:, :, 1]
    dense = [t.contiguous() for t in (q, k, v)]
    kw = dict(key_mask=mask, key_lengths=lengths)
    kw_d = dict(key_mask=mask.contiguous(), key_lengths=lengths.int())
    want = C.cross_attention_fwd(*dense, **kw_d)
    got = C.cross_attention_fwd(q, k, v, **kw)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    gw = C.cross_attention_bwd(dout.contiguous(), *dense, *want, **kw_d)
    gg = C.cross_attention_bwd(dout, q, k, v, *got, **kw)
    assert all(torch.equal(a, c) for a, c in zip(gg, gw))
    # rows 2 B off the alignment, a head_dim that is not dense, a transposed mask
    off = torch.empty(q.numel() + 1, device="cuda", dtype=q.dtype)[1:].view(dense[0].shape).copy_(q)
    wide = torch.empty((*k.shape, 2), device="cuda", dtype=k.dtype)[..., 0].copy_(k)
    mt = mask.t().contiguous().t()
    got = C.cross_attention_fwd(off, wide, v, key_mask=mt, key_lengths=lengths)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    # one prompt's states for every image
    one = kv[:1].expand(b, -1, -1, -1, -1)
    rep = one.contiguous()
    a = C.cross_attention_fwd(q, one[:, :, 0], one[:, :, 1])
    c = C.cross_attention_fwd(q, rep[:, :, 0], rep[:, :, 1])
    assert all(torch.equal(x, y) for x, y in zip(a, c))


def test_attention_infinite_masked_and_nan_seen():
    """What masked places hold changes nothing; a NaN that is seen reaches its rows only."""
    q, kv, _, _, mask, seen = _case("fp16", 2, 40, 100, 2, 2, 64, "bool", seed=9)
    clean = torch.where(seen.cuda()[:, :, None, None, None], kv, torch.zeros_like(kv))
    for bad in (float("inf"), -65504.0):
        dirty = torch.where(seen.cuda()[:, :, None, None, None], clean, torch.full_like(kv, bad))
        a = C.cross_attention_fwd(q, dirty[:, :, 0], dirty[:, :, 1], key_mask=mask)
        c = C.cross_attention_fwd(q, clean[:, :, 0], clean[:, :, 1], key_mask=mask)
        assert all(torch.equal(x, y) for x, y in zip(a, c))
    at = int(seen[0].nonzero()[0])
    dirty = clean.clone()
    dirty[0, at, 0, 1] = float("nan")       # batch 0, head 1
    a, _ = C.cross_attention_fwd(q, dirty[:, :, 0], dirty[:, :, 1], key_mask=mask)
    assert a[0, :, 1].isnan().all() and a[0, :, 0].isfinite().all() and a[1].isfinite().all()


def test_attention_autograd_and_differences():
    """The gradients that autograd returns are the op-level ones (packed, shared, frozen operands),
    and a step of the inputs changes the loss by what they say."""
    q, kv, dout, lengths, _, seen = _case("fp16", 3, 40, 77, 4, 2, 32, "lengths", seed=11)
    kv = torch.nan_to_num(kv)
    k, v = kv[:, :, 0], kv[:, :, 1]
    out, lse = C.cross_attention_fwd(q, k, v, key_lengths=lengths)
    want = C.cross_attention_bwd(dout, q, k, v, out, lse, key_lengths=lengths)
    ql, kl, vl, kvl = (t.detach().clone().requires_grad_() for t in (q, k, v, kv))
    o = C.cross_attention(ql, kl, vl, key_lengths=lengths)
    assert torch.equal(o, out)
    got = torch.autograd.grad(o, (ql, kl, vl), dout)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    dq, dkv = torch.autograd.grad(C.cross_attention_kv(ql, kvl, key_lengths=lengths), (ql, kvl), dout)
    assert torch.equal(dq, want[0]) and torch.equal(dkv[:, :, 0], want[1]) and torch.equal(dkv[:, :, 1], want[2])
    (dq,) = torch.autograd.grad(C.cross_attention(ql, k, v, key_lengths=lengths), (ql,), dout)
    assert torch.equal(dq, want[0])
    # differences of the loss sum(dout out) in 64 bits
    scale = 1.0 / math.sqrt(32)
    ref = _reference(q, k, v, dout, seen, scale)
    g = _gen(12)
    step = [torch.randn(t.shape, generator=g).double().cuda() for t in (q, k, v)]

    def loss(eps):
        x = [t.double() + eps * s for t, s in zip((q, k, v), step)]
        vis = seen.cuda()[:, None, None, :]
        kk, vv = (t.transpose(1, 2).repeat_interleave(2, 1) for t in x[1:])
        s = torch.where(vis, x[0].transpose(1, 2) @ kk.transpose(2, 3) * scale, -math.inf)
        p = torch.nan_to_num(torch.softmax(s, 3))
        return float((dout.double().transpose(1, 2) * (p @ vv)).sum())
    eps = 1e-4
    slope = (loss(eps) - loss(-eps)) / (2 * eps)
    said = sum(float((t.double() * s).sum()) for t, s in zip(want, step))
    room = sum(float((ref[n][1] * s.abs()).sum()) for n, s in zip(("dq", "dk", "dv"), step))
    assert abs(slope - said) <= room + 1e-5 * abs(slope)


def test_attention_autocast_and_other_stream():
    q, kv, dout, lengths, _, _ = _case("bf16", 2, 64, 77, 4, 4, 64, "lengths", seed=13)
    kv = torch.nan_to_num(kv)
    want, _ = C.cross_attention_fwd(q, kv[:, :, 0], kv[:, :, 1], key_lengths=lengths)
    qf, kvf = q.float().requires_grad_(), kv.float().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        o = C.cross_attention_kv(qf, kvf, key_lengths=lengths)
    assert torch.equal(o, want)
    dq, dkv = torch.autograd.grad(o, (qf, kvf), dout)
    assert dq.dtype == torch.float32 and dkv.dtype == torch.float32 and dkv.shape == kv.shape
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, _ = C.cross_attention_fwd(q, kv[:, :, 0], kv[:, :, 1], key_lengths=lengths)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o2, want)


# ---- dropout ---------------------------------------------------------------------------------
def _factor(count, p, seed):
    """Whether element i is kept, from the formula in 64-bit integers (numpy)."""
    with np.errstate(over="ignore"):
        z = np.uint64(seed) + np.arange((count + 3) // 4, dtype=np.uint64) * np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        z ^= z >> np.uint64(31)
    keep = z.view("<u2")[:count] >= int(float(np.float32(p)) * 65536)
    return torch.from_numpy(keep)


def _kept_scale(p):
    return float(np.float32(1.0) / np.float32(1.0 - float(np.float32(p))))


def _drop_ref(x, p, seed, residual=None):
    """x in memory order, CPU."""
    keep = _factor(x.numel(), p, seed).view(x.shape)
    y = torch.where(keep, x.float() * _kept_scale(p), 0.0)
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype)


def _seed(n):
    return torch.tensor([n], dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 1023, 2048, 77 * 513 + 5])
@pytest.mark.parametrize("p", [0.1, 0.5, 0.999])
def test_dropout_bits(dtype, n, p):
    g = _gen(n)
    seed = int(torch.randint(0, 2**62, (1,), generator=g))
    x = torch.randn(n, generator=g).to(DT[dtype])
    r = torch.randn(n, generator=g).to(DT[dtype])
    keep = _factor(n, p, seed)
    x[~keep & (torch.arange(n) % 3 == 0)] = float("nan")         # dropped: counts as 0
    x[~keep & (torch.arange(n) % 3 == 1)] = float("inf")
    for res in (None, r):
        want = _drop_ref(x, p, seed, res)
        got = C.dropout_fwd(x.cuda(), p, _seed(seed), residual=None if res is None else res.cuda())
        assert torch.equal(got.cpu(), want)
    # one element off the 16-B alignment
    off = torch.empty(n + 1, dtype=x.dtype, device="cuda")[1:].copy_(x)
    assert torch.equal(C.dropout_fwd(off, p, _seed(seed)).cpu(), _drop_ref(x, p, seed))


def test_dropout_layouts_and_gradients():
    g = _gen(1)
    x = torch.randn((3, 20, 6, 5), generator=g)
    p, seed = 0.25, 123456789
    for order in (torch.contiguous_format, torch.channels_last):
        xd = x.cuda().contiguous(memory_format=order).requires_grad_()
        rd = torch.randn(x.shape, generator=g).cuda().requires_grad_()     # its own layout
        y = C.dropout(xd, p, residual=rd, seed=_seed(seed))
        assert y.is_contiguous(memory_format=order)
        dy = torch.randn(x.shape, generator=g).cuda()
        gx, gr = torch.autograd.grad(y, (xd, rd), dy)

        def mem(t):
            t = t.detach().cpu()
            return t.permute(0, 2, 3, 1).contiguous() if order is torch.channels_last else t
        assert torch.equal(mem(y).contiguous(), _drop_ref(mem(xd), p, seed, mem(rd)))
        assert torch.equal(mem(gx).contiguous(), _drop_ref(mem(dy), p, seed)) and torch.equal(gr, dy)
    # neither dense nor channels last: as its dense copy
    t = x.cuda().transpose(1, 3)
    assert torch.equal(C.dropout_fwd(t, p, _seed(seed)), C.dropout_fwd(t.contiguous(), p, _seed(seed)))
    # a slope: y is linear in x
    xd = x.cuda().requires_grad_()
    y = C.dropout(xd, p, seed=_seed(seed))
    (gx,) = torch.autograd.grad(y.sum(), (xd,))
    assert torch.equal(C.dropout(torch.ones_like(x).cuda(), p, seed=_seed(seed)), gx)
    empty = C.dropout_fwd(torch.empty(0, 5, device="cuda"), p, _seed(seed))
    assert empty.shape == (0, 5)


def test_dropout_rate_and_drawn_seed():
    n, p = 1 << 20, 0.2
    torch.manual_seed(7)
    x = torch.ones(n, device="cuda")
    a, b = C.dropout(x, p), C.dropout(x, p)
    torch.manual_seed(7)
    assert torch.equal(a, C.dropout(x, p)) and not torch.equal(a, b)
    rate = float((a == 0).float().mean())
    assert abs(rate - p) < 2.0**-16 + 5 * math.sqrt(p * (1 - p) / n)
    # across the middle of the sequence of indices too: neighbours are independent
    both = float(((a[:-1] == 0) & (a[1:] == 0)).float().mean())
    assert abs(both - p * p) < 5 * math.sqrt(p * p / n) + 2.0**-15


# ---- embedding -------------------------------------------------------------------------------
@pytest.mark.parametrize("wt,ot", [("bf16", "bf16"), ("fp32", "fp32"), ("fp32", "bf16"), ("fp16", "fp16"),
                                   ("bf16", "fp32"), ("fp32", "fp16")])
@pytest.mark.parametrize("c", [1, 3, 4, 64, 260, 1023])
def test_embedding_forward_bits(wt, ot, c):
    g = _gen(c)
    v, scale, p, seed = 37, 1.7, 0.3, 987654321987
    w = torch.randn((v, c), generator=g).to(DT[wt])
    for tdt, shape in ((torch.int64, (5, 13)), (torch.int32, (1,)), (torch.int64, (0, 4))):
        t = torch.randint(0, v, shape, generator=g).to(tdt)
        want = w[t.long()].float() * np.float32(scale).item()
        got = C.embedding_fwd(t.cuda(), w.cuda(), scale=scale, out_dtype=DT[ot])
        assert got.dtype == DT[ot] and torch.equal(got.cpu(), want.to(DT[ot]))
        got = C.embedding_fwd(t.cuda(), w.cuda(), scale=scale, out_dtype=DT[ot], p_drop=p, seed=_seed(seed))
        assert torch.equal(got.cpu(), _drop_ref(want, p, seed).to(DT[ot]))


def test_embedding_outside_the_table():
    w = torch.ones((5, 8), device="cuda")
    t = torch.tensor([0, 5, -1, 4, 2**40], device="cuda")
    out = C.embedding_fwd(t, w)
    assert out[[0, 3]].eq(1).all() and out[[1, 2, 4]].isnan().all()
    dw = C.embedding_bwd(torch.ones((5, 8), device="cuda"), t, 5)
    assert torch.equal(dw.cpu(), torch.tensor([1., 0, 0, 0, 1])[:, None].expand(5, 8))


def _dw_reference(dout, tokens, v, scale, pad, p, seed):
    """(exact, bound on what fp32 sums and no rounding of the result may be off)"""
    n, c = tokens.numel(), dout.shape[-1]
    d = dout.double().view(n, c) * np.float32(scale).item()
    if p:
        d = torch.where(_factor(n * c, p, seed).view(n, c).to(d.device), d * _kept_scale(p), 0.0)
    t = tokens.long().view(-1)
    keep = (t >= 0) & (t < v)
    if pad is not None:
        keep &= t != pad
    d, t = d[keep], t[keep]
    exact = torch.zeros((v, c), dtype=torch.float64, device=d.device).index_add_(0, t, d)
    mag = torch.zeros_like(exact).index_add_(0, t, d.abs())
    count = torch.bincount(t, minlength=v).double()[:, None]
    return exact, (count + 4) * 2.0**-24 * mag


GRADS = [
    # tokens, rows, channels, dout dtype, weight dtype, padding, p
    (1, 1, 1, "fp32", "fp32", None, 0.0),
    (5, 3, 8, "fp32", "fp32", 1, 0.3),
    (64, 2, 4, "bf16", "fp32", None, 0.0),
    (65, 1, 12, "fp32", "bf16", None, 0.1),
    (1000, 7, 33, "fp32", "fp32", 0, 0.25),
    (1000, 100000, 16, "bf16", "bf16", 0, 0.0),
    (9856, 32768, 64, "fp32", "fp32", 0, 0.1),
    (16384, 300, 20, "fp16", "fp16", None, 0.0),
    (16385, 257, 260, "fp32", "fp32", None, 0.0),
    (40000, 65537, 8, "fp32", "fp32", 5, 0.0),
    (20000, 2**24 + 3, 1, "fp32", "fp32", None, 0.0),
    (140000, 3, 4, "fp32", "fp32", None, 0.0),        # long runs, two rounds of merges
    (140000, 50001, 4, "bf16", "fp32", 0, 0.0),
]


@pytest.mark.parametrize("n,v,c,gt,wt,pad,p", GRADS)
def test_embedding_gradient(n, v, c, gt, wt, pad, p):
    print(f"embedding_bwd n={n} v={v} c={c} {gt} {wt} pad={pad} p={p}", flush=True)
    g = _gen(n + v)
    u = torch.rand(n, generator=g, dtype=torch.float64)
    t = (torch.exp(u * math.log(v + 1)) - 1).long().clamp(0, v - 1)       # frequent low tokens
    t = torch.where(torch.rand(n, generator=g) < 0.05, torch.randint(-2, v + 2, (n,), generator=g), t)
    dout = torch.randn((n, c), generator=g).to(DT[gt]).cuda()
    seed, scale = 24681357, 0.8
    for tdt in (torch.int64, torch.int32):
        tokens = t.to(tdt).cuda()
        kw = dict(scale=scale, padding_idx=pad, dtype=DT[wt], p_drop=p, seed=_seed(seed) if p else None)
        dw = C.embedding_bwd(dout, tokens, v, **kw)
        torch.cuda.synchronize()
        exact, bound = _dw_reference(dout, tokens, v, scale, pad, p, seed)
        tiny = torch.finfo(DT[wt]).smallest_normal * torch.finfo(DT[wt]).eps
        assert dw.dtype == DT[wt] and dw.shape == (v, c)
        diff = (dw.double() - exact).abs()
        over = diff - (bound + HALF[DT[wt]] * exact.abs() + tiny)
        assert float(over.max()) <= 0, f"{int((over > 0).sum())} beyond the bound, worst {float(over.max()):.3e}"
        assert torch.equal(dw, C.embedding_bwd(dout, tokens, v, **kw))
        if pad is not None:
            assert not dw[pad].any()


@pytest.mark.parametrize("n,v,c", [(17, 2, 70), (255, 1, 64), (256, 3, 65), (257, 1000, 130), (512, 2, 3),
                                   (512, 2**18, 8), (511, 2**18 + 1, 8), (513, 5, 64), (300, 40000, 1)])
@pytest.mark.parametrize("gt,wt,pad", [("fp32", "fp32", None), ("bf16", "bf16", 0), ("fp16", "fp32", 1)])
def test_embedding_gradient_few_tokens(n, v, c, gt, wt, pad):
    """The form of one launch and its border: runs over several waves, rows that no token names, odd
    widths, tokens outside the table."""
    print(f"embedding_bwd n={n} v={v} c={c} {gt} {wt} pad={pad}", flush=True)
    pad = pad if pad is None or pad < v else None
    g = _gen(n * 31 + v)
    t = torch.randint(0, v, (n,), generator=g)
    t = torch.where(torch.rand(n, generator=g) < 0.05, torch.randint(-2, v + 2, (n,), generator=g), t).cuda()
    dout = torch.randn((n, c), generator=g).to(DT[gt]).cuda()
    for p in (0.0, 0.3):
        dw = C.embedding_bwd(dout, t, v, scale=0.8, padding_idx=pad, dtype=DT[wt], p_drop=p,
                             seed=_seed(77) if p else None)
        torch.cuda.synchronize()
        exact, bound = _dw_reference(dout, t, v, 0.8, pad, p, 77)
        tiny = torch.finfo(DT[wt]).smallest_normal * torch.finfo(DT[wt]).eps
        over = (dw.double() - exact).abs() - (bound + HALF[DT[wt]] * exact.abs() + tiny)
        assert float(over.max()) <= 0, f"{int((over > 0).sum())} beyond the bound, worst {float(over.max()):.3e}"


def test_embedding_gradient_without_tokens():
    dw = C.embedding_bwd(torch.empty((0, 5), device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), 9)
    assert dw.shape == (9, 5) and not dw.any()


def test_embedding_autograd():
    g = _gen(2)
    w = torch.randn((50, 24), generator=g).cuda().requires_grad_()
    t = torch.randint(0, 50, (4, 9), generator=g).cuda()
    dout = torch.randn((4, 9, 24), generator=g).cuda()
    out = C.embedding(t, w, scale=2.0, padding_idx=3, p_drop=0.4, seed=_seed(5), out_dtype=torch.bfloat16)
    assert out.dtype == torch.bfloat16
    (dw,) = torch.autograd.grad(out, (w,), dout.bfloat16())
    assert dw.dtype == torch.float32
    want = C.embedding_bwd(dout.bfloat16(), t, 50, scale=2.0, padding_idx=3, p_drop=0.4, seed=_seed(5),
                           dtype=torch.float32)
    assert torch.equal(dw, want)
    # a slope: out is linear in the weight
    w2 = torch.randn((50, 24), generator=g).cuda()
    w2[3] = 0
    o = C.embedding_fwd(t, w2, scale=2.0, p_drop=0.4, seed=_seed(5))
    g32 = C.embedding_bwd(dout, t, 50, scale=2.0, padding_idx=3, p_drop=0.4, seed=_seed(5))
    a, b = float((o.double() * dout.double()).sum()), float((w2.double() * g32.double()).sum())
    assert abs(a - b) <= 2.0**-20 * float((o.double() * dout.double()).abs().sum())
    assert torch.equal(C.embedding(t, w2, scale=2.0, p_drop=0.4, training=False), C.embedding_fwd(t, w2, scale=2.0))


# ---- captured ----------------------------------------------------------------------------------
def test_captured_step_replays():
    """Forward and backward of all three in one HIP graph: every replay equals the eager calls on
    the same inputs, with eager work and synchronisation between."""
    g = _gen(21)
    tokens = torch.randint(0, 500, (8, 77), generator=g).cuda()
    table = torch.randn((500, 128), generator=g).cuda()
    q = torch.randn((8, 64, 2, 64), generator=g).bfloat16().cuda()
    dout = torch.randn((8, 64, 2, 64), generator=g).bfloat16().cuda()
    lengths = torch.randint(0, 78, (8,), generator=g).int().cuda()
    seed = _seed(99)

    def step():
        e = C.embedding_fwd(tokens, table, scale=2.0, p_drop=0.1, seed=seed, out_dtype=torch.bfloat16)
        s = C.dropout_fwd(e, 0.2, seed)
        k = s.view(8, 77, 2, 64)
        out, lse = C.cross_attention_fwd(q, k, k, key_lengths=lengths)
        dq, dk, dv = C.cross_attention_bwd(dout, q, k, k, out, lse, key_lengths=lengths)
        ds = C.dropout_bwd((dk + dv).view(8, 77, 128), 0.2, seed)
        dw = C.embedding_bwd(ds, tokens, 500, scale=2.0, padding_idx=0, p_drop=0.1, seed=seed,
                             dtype=torch.float32)
        return e, s, out, lse, dq, dk, dv, dw
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=g).bfloat16())
        tokens.copy_(torch.randint(0, 500, (8, 77), generator=g))
        lengths.copy_(torch.randint(0, 78, (8,), generator=g).int())
        seed.fill_(1000 + i)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


# ---- the native calls and the general way -------------------------------------------------------
def test_fast_calls_and_the_general_way_agree(monkeypatch):
    """Both ways to a launch give the same bits, and the operands that need no conversion take the
    native one."""
    fast = C._fast()
    assert not isinstance(fast, C._General)
    q, kv, dout, lengths, mask, _ = _case("bf16", 3, 40, 77, 4, 2, 64, "both", seed=31)
    kv = torch.nan_to_num(kv)
    k, v = kv[:, :, 0], kv[:, :, 1]
    g = _gen(32)
    x = torch.randn((6, 33), generator=g).cuda()
    img = torch.randn((2, 8, 4, 4), generator=g).cuda().contiguous(memory_format=torch.channels_last)
    table = torch.randn((20, 24), generator=g).cuda()
    tokens = torch.randint(0, 20, (4, 7), generator=g).cuda()
    grad = torch.randn((4, 7, 24), generator=g).cuda()

    def calls():
        kw = dict(key_lengths=lengths, key_mask=mask)
        out, lse = C.cross_attention_fwd(q, k, v, **kw)
        dkv = torch.empty_like(kv)
        return [out, lse, *C.cross_attention_bwd(dout, q, k, v, out, lse, **kw),
                *C.cross_attention_fwd(q, k, v, scale=0.3),
                C._attention_bwd(dout, q, k, v, out, lse, lengths, mask, None, None, None)[0],
                *C._attention_bwd(dout, q, k, v, out, lse, lengths, mask, None, dkv[:, :, 0], dkv[:, :, 1]), dkv,
                C.dropout_fwd(x, 0.3, _seed(5)), C.dropout_fwd(img, 0.3, _seed(5), residual=img),
                C.embedding_fwd(tokens, table, scale=2.0, p_drop=0.2, seed=_seed(6), out_dtype=torch.bfloat16),
                C.embedding_fwd(tokens.int(), table),
                C.embedding_bwd(grad, tokens, 20, scale=2.0, padding_idx=3, p_drop=0.2, seed=_seed(6)),
                C.embedding_bwd(grad, tokens, 20, dtype=torch.bfloat16)]
    assert fast.attention_fwd(q, k, v, lengths, mask, None) is not None
    assert fast.attention_fwd(q[:2], k, v, None, None, None) is None                   # another batch
    assert fast.attention_fwd(q, k, v, lengths.long(), None, None) is None             # int64 is converted
    assert fast.dropout(img, 0.3, _seed(5), img) is not None
    assert fast.dropout(img, 1.0, _seed(5), None) is None and fast.dropout(img, 0.3, None, None) is None
    assert fast.embedding_bwd(grad, tokens, 20, 1.0, 20, 0.0, None, None) is None      # padding outside the rows
    here = calls()
    monkeypatch.setattr(C, "_FAST", C._General())
    there = calls()
    assert len(here) == len(there)
    for a, b in zip(here, there):
        assert a.dtype == b.dtype and a.stride() == b.stride() and torch.equal(a, b)


def test_fast_calls_keep_to_the_current_stream_and_free_what_they_make():
    q = torch.randn((2, 64, 2, 64), device="cuda").bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big = torch.randn((1 << 24,), device="cuda")
        x = (big * 0 + 2).view(-1)                 # work in flight that the call has to stand behind
        y = C.dropout_fwd(x, 0.5, _seed(3))
    torch.cuda.current_stream().wait_stream(side)
    assert bool(((y == 0) | (y == 4)).all()) and bool(y.any())
    del x, y, big
    torch.cuda.synchronize()
    for _ in range(3):
        C.cross_attention_fwd(q, q, q)
    before = torch.cuda.memory_allocated()
    for _ in range(20):
        o, lse = C.cross_attention_fwd(q, q, q)
        C.cross_attention_bwd(q, q, q, q, o, lse)
    del o, lse
    assert torch.cuda.memory_allocated() == before
