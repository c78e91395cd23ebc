"""The text-conditioned U-Net: prompts kept for sampling against training, and the captured step."""
from __future__ import annotations

import pytest
import torch

from conftest import dpa_mod
from test_gpu_text_unet import _config, _images, _model, _text, _tokens

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


@pytest.mark.parametrize("scaling", ["current", "delayed"])
def test_captured_steps_are_the_eager_ones_to_the_bit(scaling):
    g = torch.Generator().manual_seed(11)
    data = [(_images(8, g), torch.randint(0, 100, (8,), generator=g).cuda(), _images(8, g), _tokens(8, 12, g))
            for _ in range(4)]

    def state():
        s = T.TrainState(_config(fp8_scaling_type=scaling), 8, max_t=100, text=_text(), prompt_length=12,
                         fixed_noise=True, ema_beta=0.9, seed=1)
        s.set_batch(*data[0])
        return s

    def walk(s, step):
        losses = []
        for i in range(6):
            s.set_batch(*data[i % 4])
            s.loss_acc.zero_()
            step()
            torch.cuda.synchronize()
            losses.append(float(s.loss_acc))
        return losses
    a, b = state(), state()
    before = a.model.text.weight.detach().clone()
    a.capture(warmup=3)
    for _ in range(3):
        b.eager_step()
    assert walk(a, a.replay) == walk(b, b.eager_step)
    for (n, p), q in zip(a.model.named_parameters(), b.model.parameters()):
        assert torch.equal(p, q), n
    dw = a.model.text.weight.grad
    assert dw is not None and bool(dw.isfinite().all()) and bool(dw.any()) and not dw[0].any()
    assert bool((a.model.text.weight[1:] != before[1:]).any())
