"""The text-conditioned U-Net: the operators of ``conditioning`` as the model runs them."""
from __future__ import annotations

import importlib.util
import math
import os

import pytest
import torch

from conftest import ROOT, dpa_mod

pytestmark = pytest.mark.gpu

C = dpa_mod("conditioning")
U = dpa_mod("unet")
X = dpa_mod("text_unet")
T = dpa_mod("trainer")


def _config(**kw):
    """Every convolution and projection of the base model on this framework's kernels, which give the
    same bits each time (the library's convolutions do not)."""
    return U.UNetConfig(**{**dict(in_channels=3, base_hidden=128, scales=[1, 2], n_heads=2, p_drop=0.0,
                                  attn_resolutions=[16], in_resolution=16, n_resblocks=2,
                                  fp8_convs_enabled=True, fp8_scaling_type="current",
                                  fp8_all_convs=True, fp8_linears=True), **kw})


def _text(**kw):
    return X.TextConfig(**{**dict(vocab=50, width=96, p_drop=0.0), **kw})


def _tokens(b, length, g):
    t = torch.randint(1, 50, (b, length), generator=g)
    ends = torch.randint(0, length + 1, (b, 1), generator=g)
    ends[0], ends[-1] = length, 0              # a full prompt and a dropped one
    return torch.where(torch.arange(length) < ends, t, 0).cuda()


def _model(seed=0, text=None, live=True, **kw):
    torch.manual_seed(seed)
    m = X.TextUNet(_config(**kw), text or _text()).to(memory_format=torch.channels_last).cuda()
    if live:        # output weights that are not zero, so that every part reaches the loss
        g = torch.Generator().manual_seed(seed + 1)
        for p in m.parameters():
            if not p.any() and p.ndim > 1:
                p.data.copy_(torch.randn(p.shape, generator=g) * 0.05)
    return m


def _images(b, g, size=16):
    return torch.randn((b, 3, size, size), generator=g).cuda().contiguous(memory_format=torch.channels_last)


def test_without_prompt_and_at_the_start_it_is_the_base_model():
    g = torch.Generator().manual_seed(3)
    m = _model(live=False)
    base = U.UNet(_config()).to(memory_format=torch.channels_last).cuda()
    missing = base.load_state_dict(m.state_dict(), strict=False)
    assert not missing.missing_keys
    assert all(k.startswith(("text.", "cross.")) for k in missing.unexpected_keys)
    for mod in (m, base):
        mod.eval()
        torch.manual_seed(9)
        with torch.no_grad():
            mod.out[-1].weight.normal_()       # (the base model's output starts at zero too)
    x, t = _images(3, g), torch.tensor([1, 50, 99], device="cuda")
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        want = base(x, t)
        assert torch.equal(m(x, t), want)
        assert torch.equal(m(x, t, _tokens(3, 20, g)), want)     # zero output projections


def test_block_against_64_bits():
    """The block against its formula in 64 bits from the bf16 numbers that its products take. Each of
    the six roundings to bf16 on the way (norm, q, kv, attention, out, sum) is at most 2^-8 of a
    magnitude that the next product's operand norms bound."""
    g = torch.Generator().manual_seed(5)
    text = _text()
    torch.manual_seed(4)
    block = X.CrossAttentionBlock(64, text, 2).cuda()
    with torch.no_grad():
        block.out.weight.normal_(std=0.1)
    x = torch.randn((2, 64, 6, 5), generator=g).bfloat16().cuda().contiguous(memory_format=torch.channels_last)
    states = torch.randn((2, 11, 96), generator=g).bfloat16().cuda()
    mask = (torch.rand((2, 11), generator=g) < 0.7).cuda()
    mask[1] = False
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        y = block(x, block.project(states), mask)
    assert y.shape == x.shape and y.is_contiguous(memory_format=torch.channels_last)

    def w(p):
        return p.detach().bfloat16().double()
    seq = x.permute(0, 2, 3, 1).reshape(2, 30, 64).double()
    n = torch.nn.functional.layer_norm(seq, (64,), block.norm.weight.double(), block.norm.bias.double())
    q = (n @ w(block.q.weight).T).view(2, 30, 2, 32)
    kv = (states.double() @ w(block.kv.weight).T).view(2, 11, 2, 2, 32)
    k, v = kv.unbind(2)
    s = torch.einsum("bqhd,bkhd->bhqk", q, k) / math.sqrt(32)
    s = torch.where(mask[:, None, None, :], s, -math.inf)
    p = torch.nan_to_num(torch.softmax(s, 3))
    o = torch.einsum("bhqk,bkhd->bqhd", p, v).reshape(2, 30, 64)
    want = seq + o @ w(block.out.weight).T
    u = 2.0**-8
    # |ds| <= scale (|dq| |k| + |q| |dk|) with dq, dk of three and one roundings
    ds = 4 * u * torch.einsum("bqhd,bkhd->bhqk", q.abs() + u, k.abs() + u) / math.sqrt(32)
    ds = ds + 2 * u * torch.einsum("bqc,hdc,bkhd->bhqk", n.abs(), w(block.q.weight).abs().view(2, 32, 64), k.abs()) / math.sqrt(32)
    rel = 2 * torch.where(mask[:, None, None, :], ds, 0.0).amax(3, keepdim=True)
    do = torch.einsum("bhqk,bkhd->bqhd", p * (rel.exp() - 1 + 2 * u), v.abs()).reshape(2, 30, 64)
    do = do + 2 * u * o.abs()
    tol = do @ w(block.out.weight).abs().T + 2 * u * (o.abs() @ w(block.out.weight).abs().T) + 2 * u * want.abs()
    got = y.permute(0, 2, 3, 1).reshape(2, 30, 64).double()
    assert bool(((got - want).abs() <= tol).all())
    assert torch.equal(got[1], seq[1])                # a prompt without tokens leaves the image alone


def test_kept_prompt_is_the_prompt():
    g = torch.Generator().manual_seed(7)
    m = _model().eval()
    x, t, tokens = _images(4, g), torch.tensor([3, 10, 40, 90], device="cuda"), _tokens(4, 20, g)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        want = m(x, t, tokens)
        plain = m(x, t)
        assert not torch.equal(want, plain)
        m.keep_prompt(tokens)
        assert torch.equal(m(x, t), want)
        other = _tokens(4, 9, g)
        assert not torch.equal(m(x, t, other), want)          # a call's own prompt comes first
        m.keep_prompt(None)
        assert torch.equal(m(x, t), plain)
        m.prompt = tokens
        assert torch.equal(m(x, t), want)


def test_gradients_reach_the_text():
    g = torch.Generator().manual_seed(8)
    m = _model(text=_text(p_drop=0.1), p_drop=0.1).train()
    x, t, tokens = _images(4, g), torch.tensor([3, 10, 40, 90], device="cuda"), _tokens(4, 20, g)

    def loss():
        torch.manual_seed(17)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            return m(x, t, tokens).float().square().mean()
    loss().backward()
    grads = {n: p.grad.clone() for n, p in m.named_parameters()}
    dw = grads["text.weight"]
    used = torch.zeros(50, dtype=torch.bool, device="cuda")
    used[tokens.flatten()] = True
    used[0] = False
    assert dw.dtype == torch.float32 and bool((dw[used].abs().amax(1) > 0).all()) and not dw[~used].any()
    for n, v in grads.items():
        assert v.isfinite().all(), n
        if n.startswith("cross."):
            assert v.any(), n
    m.zero_grad()
    loss().backward()
    for n, p in m.named_parameters():
        if n.startswith(("cross.", "text.")):
            assert torch.equal(p.grad, grads[n]), n            # deterministic


def test_captured_training_step():
    """Replays of the captured step equal eager steps, prompts written between them."""
    g = torch.Generator().manual_seed(11)
    data = [(_images(8, g), torch.randint(0, 100, (8,), generator=g).cuda(), _images(8, g), _tokens(8, 12, g))
            for _ in range(4)]

    def state():
        return T.TrainState(_config(), 8, max_t=100, text=_text(), prompt_length=12, fixed_noise=True,
                            ema_beta=0.9, seed=1)

    def walk(s, step):
        out = []
        for i in range(6):
            x, t, eps, tokens = data[i % 4]
            s.set_batch(x, t, eps, tokens)
            s.loss_acc.zero_()
            step()
            torch.cuda.synchronize()
            out.append(float(s.loss_acc))
        return out
    a = state()
    a.set_batch(*data[0])
    a.capture(warmup=3)
    replayed = walk(a, a.replay)
    b = state()
    b.set_batch(*data[0])
    for _ in range(3):
        b.eager_step()
    eager = walk(b, b.eager_step)
    for x, y in zip(replayed, eager):
        assert abs(x - y) <= 1e-3 * abs(y)
    assert replayed[-1] < replayed[0]
    assert a.model.text.weight.grad is None or a.model.text.weight.grad.isfinite().all()
    assert not a.model.text.weight[0].any()                   # the padding learns nothing


def test_example_runs():
    spec = importlib.util.spec_from_file_location("text_to_image", os.path.join(ROOT, "examples", "text_to_image.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    losses = ex.main(["--steps", "100", "--batch", "16", "--max-t", "20", "--prompts", "red disc", ""])
    assert len(losses) == 2 and losses[1] < losses[0]
