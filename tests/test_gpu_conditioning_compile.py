"""The conditioning operators and the text-conditioned U-Net under torch.compile: they run between the
graphs, as the framework's other launches do, and give the eager numbers."""
from __future__ import annotations

import warnings

import pytest
import torch
import torch._dynamo

from conftest import dpa_mod

pytestmark = pytest.mark.gpu

C = dpa_mod("conditioning")
U = dpa_mod("unet")
X = dpa_mod("text_unet")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _compiled(fn):
    torch._dynamo.reset()
    return torch.compile(fn, backend="aot_eager")


def test_operators_compile():
    g = _gen(1)
    tokens = torch.randint(0, 30, (3, 20), generator=g).cuda()
    table = torch.randn((30, 64), generator=g).cuda()
    q = torch.randn((3, 40, 2, 32), generator=g).bfloat16().cuda()
    seed = torch.tensor([77], device="cuda")

    def f(tokens, table, q):
        e = C.embedding(tokens, table, scale=2.0, padding_idx=0, p_drop=0.1, seed=seed, out_dtype=torch.bfloat16)
        k = e.view(3, 20, 2, 32)
        o = C.cross_attention(q * 2, k, k, key_mask=tokens != 0)
        kv = torch.stack((k, k), 2)
        o = o + C.cross_attention_kv(q, kv, key_mask=tokens != 0)
        return C.dropout(o * 3, 0.2, residual=q, seed=seed)

    def run(fn):
        a, b = table.clone().requires_grad_(), q.clone().requires_grad_()
        y = fn(tokens, a, b)
        y.float().square().sum().backward()
        return y.detach(), a.grad, b.grad
    want = run(f)
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        fn = _compiled(f)
        for _ in range(2):
            assert all(torch.equal(x, y) for x, y in zip(run(fn), want))
    assert not [str(w.message) for w in seen if "dpa_fast_calls" in str(w.message) or "builtin" in str(w.message)]
    with torch.no_grad():
        y = f(tokens, table, q)
        assert torch.equal(_compiled(f)(tokens, table, q), y)


def test_text_unet_compiles():
    cfg = U.UNetConfig(in_channels=3, base_hidden=128, scales=[1, 2], n_heads=2, p_drop=0.0, attn_resolutions=[16],
                       in_resolution=16, n_resblocks=2, fp8_convs_enabled=True, fp8_scaling_type="current",
                       fp8_all_convs=True, fp8_linears=True)
    torch.manual_seed(2)
    m = X.TextUNet(cfg, X.TextConfig(vocab=50, width=96, p_drop=0.0)).to(memory_format=torch.channels_last).cuda()
    g = _gen(3)
    for p in m.parameters():
        if not p.any() and p.ndim > 1:
            p.data.copy_(torch.randn(p.shape, generator=g) * 0.05)
    x = torch.randn((2, 3, 16, 16), generator=g).cuda().contiguous(memory_format=torch.channels_last)
    t = torch.tensor([3, 70], device="cuda")
    tokens = torch.randint(0, 50, (2, 12), generator=g).cuda()

    def step(model):
        m.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = model(x, t, tokens)
        y.float().square().mean().backward()
        return [y.detach()] + [p.grad.clone() for p in m.parameters()]
    want = step(m)
    torch._dynamo.reset()
    fn = torch.compile(m, backend="aot_eager")
    for _ in range(2):
        for a, b in zip(step(fn), want):
            assert torch.equal(a, b)
