"""How far cross attention's results may be off as a whole: the formula in 64 bits with the expected
square of each element's error, and a comparison of norms.

A rounding to the operands' type is taken as independent and uniform in half a step, so a number x
carries the variance r2 x^2, r2 = u^2 / 3 (u = finfo.eps / 2), and where the type is fp16 at least
f2 = (2^-25)^2 / 3, half of its subnormal step. The roundings of a call are
  P for its product with v, out, P and dS for their products in the backward, dq, dk, dv
and D = rowsum(dout out) takes out as rounded. Through the formulas:
  var out = sum_k (r2 P^2 + f2) v^2 + R(out)          R(x) = r2 x^2 + f2
  var D   = sum_d dout^2 var out
  var dq  = scale^2 (sum_k e2 k^2 + var D (sum_k P k)^2) + R(dq)
  var dk  = scale^2 sum_rows (e2 + P^2 var D) q^2 + R(dk)
  var dv  = sum_rows r2 P^2 dout^2 + R(dv)
with e2 = r2 dS^2 + (P rho)^2 (dP^2 + D^2) + (2^-22 P sum |dout v|)^2 for dS: its rounding and what the
fp32 numbers behind it are off by, rho = 2^-20 (1 + max |score| / 8) for the exponent's argument. dS has
no absolute term: the kernels scale it. An error of a uniform rounding is at most sqrt(3) of its
deviation and the mean over mantissas is 0.72 of it, so a tensor's squared error beyond 4 times the sum of
the variances, or a head's beyond 9 times, is not rounding.
"""
from __future__ import annotations

import math

import torch

HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TENSOR, HEAD = 2.0, 3.0         # deviations


def _heads(t, n=1):
    return t.double().transpose(1, 2).repeat_interleave(n, 1)


def _out(t):
    return t.transpose(1, 2)


def reference(q, k, v, dout, seen, scale):
    """{name: (exact, variance)}, laid out as the operands (v and k may hold anything where not seen)."""
    u = HALF[q.dtype]
    r2 = u * u / 3
    f2 = (2.0**-25) ** 2 / 3 if q.dtype == torch.float16 else 0.0
    b, _, h, d = q.shape
    lk, kvh = k.shape[1:3]
    rep = h // kvh
    vis = seen.to(q.device)[:, None, None, :]
    q_, do = _heads(q), _heads(dout)
    k_, v_ = (torch.where(vis.transpose(2, 3), _heads(t, rep), 0.0) for t in (k, v))
    x = torch.where(vis, (q_ @ k_.transpose(2, 3).contiguous()) * scale, -math.inf)
    top = x.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(x - top)
    tot = e.sum(3, keepdim=True)
    p = e / torch.where(tot == 0, 1.0, tot)
    rho = 2.0**-20 * (1 + torch.where(vis, x.abs(), 0.0).amax(3, keepdim=True) / 8)
    o = p @ v_
    var_o = (r2 * p * p + torch.where(vis, f2, 0.0)) @ (v_ * v_) + r2 * o * o + f2
    dp = do @ v_.transpose(2, 3).contiguous()
    dpm = do.abs() @ v_.abs().transpose(2, 3).contiguous()
    dd = (do * o).sum(3, keepdim=True)
    var_d = (do * do * var_o).sum(3, keepdim=True)
    ds = p * (dp - dd)
    e2 = r2 * ds * ds + (p * rho) ** 2 * (dp * dp + dd * dd) + (2.0**-22 * p * dpm) ** 2
    dq = scale * (ds @ k_)
    var_q = scale**2 * (e2 @ (k_ * k_) + var_d * (p @ k_) ** 2) + r2 * dq * dq + f2

    def shared(t):
        return t.reshape(b, kvh, rep, lk, d).sum(2)
    dk = shared(scale * (ds.transpose(2, 3).contiguous() @ q_))
    var_k = shared(scale**2 * ((e2 + p * p * var_d).transpose(2, 3).contiguous() @ (q_ * q_))) + r2 * dk * dk + f2
    dv = shared(p.transpose(2, 3).contiguous() @ do)
    var_v = shared(((r2 + rho * rho) * p * p).transpose(2, 3).contiguous() @ (do * do)) + r2 * dv * dv + f2
    return {n: (_out(a), _out(c)) for n, a, c in
            (("out", o, var_o), ("dq", dq, var_q), ("dk", dk, var_k), ("dv", dv, var_v))}


def excess(got, ref):
    """{name: (a tensor's, its worst head's error in the deviations allowed)}: above 1 is too far off.
    Heads are counted from 64 numbers on."""
    res = {}
    for name, t in got.items():
        exact, var = ref[name]
        assert t.shape == exact.shape, name
        err = (t.double() - exact) ** 2
        assert bool(err.isfinite().all()), f"{name} is not finite"

        def ratio(e, w):
            return float((e / torch.where(w == 0, 1.0, w)).masked_fill((e > 0) & (w == 0), math.inf).max())
        whole = ratio(err.sum(), var.sum()) if err.numel() else 0.0
        head = 0.0
        if err.shape[1] * err.shape[3] >= 64 and err.numel():
            head = ratio(err.sum((1, 3)), var.sum((1, 3)))
        res[name] = (math.sqrt(whole) / TENSOR, math.sqrt(head) / HEAD)
    return res


def check(got, ref):
    worst = {n: e for n, e in excess(got, ref).items() if max(e) > 1}
    assert not worst, f"beyond the deviations allowed (tensor, worst head): {worst}"


def inputs(dtype, b, lq, lk, h, kvh, d, seed, offset=0.0, dout_std=1.0, q_std=1.0):
    """q, kv, dout on the CPU; offset: a mean of keys and values (and half of it of dout's deviation),
    with which a missing D or a missing key shows in every sum."""
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn((b, lq, h, d), generator=g) * q_std).to(dtype)
    kv = (torch.randn((b, lk, 2, kvh, d), generator=g) + offset).to(dtype)
    dout = ((torch.randn((b, lq, h, d), generator=g) + offset / 2) * dout_std).to(dtype)
    return q, kv, dout


def simulate(q, k, v, dout, seen, scale, scaled=True, drop=0, no_d=False):
    """The kernels' roundings on the CPU. scaled: P and dS are scaled before they are rounded. Faults to
    plant: drop (as many keys at the end are left out of the sums over keys), no_d."""
    dt = q.dtype
    up = 2.0**14 if scaled and dt == torch.float16 else 1.0
    b, _, h, d = q.shape
    lk, kvh = k.shape[1:3]
    rep = h // kvh
    vis = seen[:, None, None, :]
    q_, do = _heads(q), _heads(dout)
    k_, v_ = (torch.where(vis.transpose(2, 3), _heads(t, rep), 0.0) for t in (k, v))
    x = torch.where(vis, (q_ @ k_.transpose(2, 3)) * scale, -math.inf)
    top = x.amax(3, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    tot = e.sum(3, keepdim=True)
    tot = torch.where(tot == 0, 1.0, tot)
    p = e / tot
    n = lk - drop
    o = ((e.to(dt).double() / tot)[..., :n] @ v_[:, :, :n]).to(dt)
    dd = 0.0 if no_d else (do * o.double()).sum(3, keepdim=True)
    ds = p * (do @ v_.transpose(2, 3) - dd)
    if up > 1.0:
        up_s = 2.0 ** torch.floor(11 - torch.log2(ds.abs().amax(3, keepdim=True).clamp_min(2.0**-60)))
        ds_q, ds_k = (ds * up_s).to(dt).double() / up_s, None
        up_k = 2.0 ** torch.floor(11 - torch.log2(ds.abs().amax(2, keepdim=True).clamp_min(2.0**-60)))
        ds_k = (ds * up_k).to(dt).double() / up_k
    else:
        ds_q = ds_k = ds.to(dt).double()

    def shared(t):
        return _out(t.view(b, kvh, rep, lk, d).sum(2).to(dt))
    return dict(out=_out(o), dq=_out((scale * (ds_q[..., :n] @ k_[:, :, :n])).to(dt)),
                dk=shared(scale * (ds_k.transpose(2, 3) @ q_)),
                dv=shared((p * up).to(dt).double().transpose(2, 3) @ do / up))
