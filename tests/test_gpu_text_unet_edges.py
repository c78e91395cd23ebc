"""The text-conditioned U-Net: prompts kept for sampling against training."""
from __future__ import annotations

import pytest
import torch

from conftest import dpa_mod
from test_gpu_text_unet import _images, _model, _text, _tokens

pytestmark = pytest.mark.gpu

T = dpa_mod("trainer")


def _loss(m, x, t):
    torch.manual_seed(17)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        return m(x, t).float().square().mean()


def test_training_takes_the_prompt_whatever_is_kept_for_sampling():
    g = torch.Generator().manual_seed(8)
    m = _model(text=_text(p_drop=0.1)).train()
    x, t, tokens = _images(4, g), torch.tensor([3, 10, 40, 90], device="cuda"), _tokens(4, 20, g)
    m.prompt = tokens
    want = _loss(m, x, t)
    want.backward()
    grads = {n: p.grad.clone() for n, p in m.named_parameters() if n.startswith(("text.", "cross."))}
    m.zero_grad()
    m.keep_prompt(_tokens(4, 9, g))
    loss = _loss(m, x, t)
    assert torch.equal(loss, want)
    loss.backward()
    assert grads["text.weight"].any()
    for n, p in m.named_parameters():
        if n in grads:
            assert torch.equal(p.grad, grads[n]), n
    with torch.no_grad():       # and sampling the kept one, in either mode
        for mode in (True, False):
            m.train(mode).keep_prompt(_tokens(4, 9, g))
            a = _loss(m, x, t)
            m.keep_prompt(None)
            assert not torch.equal(a, _loss(m, x, t))


def test_a_prompt_kept_in_training_mode_is_kept_without_dropout():
    g = torch.Generator().manual_seed(9)
    m = _model(text=_text(p_drop=0.5))
    x, t, tokens = _images(4, g), torch.tensor([3, 10, 40, 90], device="cuda"), _tokens(4, 20, g)
    with torch.no_grad():
        m.eval().keep_prompt(tokens)
        want = _loss(m, x, t)
        m.train().keep_prompt(tokens)
        assert m.training and m.text.training
        assert torch.equal(_loss(m.eval(), x, t), want)
