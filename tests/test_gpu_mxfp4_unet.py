"""The text-conditioned U-Net on 4-bit operands: the operators of ``mxfp4`` together, as training and sampling
run them. Each operator is held to its formula in 64 bits elsewhere; here their chain is held to the bit."""
from __future__ import annotations

import importlib.util
import os
import warnings

import pytest
import torch
import torch._dynamo

from conftest import ROOT, dpa_mod
from test_gpu_text_unet import _config, _images, _model, _text, _tokens

pytestmark = pytest.mark.gpu

C = dpa_mod("conditioning")
G = dpa_mod("gn_silu")
LN = dpa_mod("layer_norm")
M = dpa_mod("mxfp4")
T = dpa_mod("trainer")
X = dpa_mod("text_unet")


@pytest.fixture
def seeds(monkeypatch):
    """The forward's seeds from a tensor that tests write, not from torch's generator."""
    kept = torch.arange(1, 65, device="cuda") * 7919

    def fill(self, device, count):
        assert count <= kept.numel()
        self.seeds, self.next = kept[:count], 0
    monkeypatch.setattr(G.DropoutSeeds, "fill", fill)

    def none_left(device):
        raise AssertionError("a seed that the forward did not count")
    monkeypatch.setattr(G, "new_dropout_seed", none_left)
    return kept


def _four(**kw):
    return _text(mxfp4=True, **kw)


def _block(seed=4):
    torch.manual_seed(seed)
    block = X.CrossAttentionBlock(64, _four(), 2).cuda()
    with torch.no_grad():
        block.out.weight.normal_(std=0.1)
    return block


def _inputs(g):
    x = torch.randn((2, 64, 6, 5), generator=g).bfloat16().cuda().contiguous(memory_format=torch.channels_last)
    states = torch.randn((2, 11, 96), generator=g).bfloat16().cuda()
    mask = (torch.rand((2, 11), generator=g) < 0.7).cuda()
    mask[1] = False
    return x, states, mask


def test_block_is_the_chain_of_its_operators():
    block = _block()
    x, states, mask = _inputs(torch.Generator().manual_seed(5))
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        kv = M.quantize_mxfp4(block.project(states))
        y = block(x, kv, mask)
        seq = x.permute(0, 2, 3, 1).reshape(2, 30, 64)
        n = LN.layer_norm_bf16(seq, block.norm)
    q = M.linear_mxfp4_fwd(n, block.q.weight).view(2, 30, 2, 32)
    k = M.linear_mxfp4_fwd(states, block.kv.weight).view(2, 11, 2, 2, 32)
    assert k.dtype == torch.bfloat16
    o, lse = M.cross_attention_mxfp4_fwd(q, M.quantize_mxfp4(k), key_mask=mask)
    assert bool((lse[1] == -torch.inf).all()) and not o[1].any()
    o = M.linear_mxfp4_fwd(o.view(2, 30, 64), block.out.weight)
    want = (seq + o).reshape(2, 6, 5, 64).permute(0, 3, 1, 2)
    assert torch.equal(y, want) and y.is_contiguous(memory_format=torch.channels_last)
    assert torch.equal(y[1], x[1])
    # laid out once, the weights give the same; writing them does not reach the kept ones
    for layer in (block.q, block.out):
        layer.keep_weight()
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(block(x, kv, mask), y)
        block.out.weight.mul_(2)
        assert torch.equal(block(x, kv, mask), y)
        for layer in (block.q, block.out):
            layer.keep_weight(False)
        assert not torch.equal(block(x, kv, mask), y)


def test_gradients_of_a_block_are_the_chain(seeds):
    block = _block().train()
    x, states, mask = _inputs(torch.Generator().manual_seed(6))
    mask[1, :3] = True
    x.requires_grad_()
    states.requires_grad_()
    G.DROPOUT_SEEDS.fill("cuda", 3)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = block(x, block.project(states), mask)
    G.DROPOUT_SEEDS.clear()
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(7)).bfloat16().cuda().contiguous(
        memory_format=torch.channels_last)
    y.backward(dy)
    kv, k_kept = M.linear_mxfp4_train_fwd(states.detach(), block.kv.weight.detach())
    seq = x.detach().permute(0, 2, 3, 1).reshape(2, 30, 64)
    with torch.no_grad():
        n = LN.layer_norm_bf16(seq, block.norm)
    q, q_kept = M.linear_mxfp4_train_fwd(n, block.q.weight.detach())
    q, kv = q.view(2, 30, 2, 32), kv.view(2, 11, 2, 2, 32)
    o, lse = C.cross_attention_fwd(q, kv[:, :, 0], kv[:, :, 1], key_mask=mask)
    _, o_kept = M.linear_mxfp4_train_fwd(o.view(2, 30, 64), block.out.weight.detach())
    d = dy.permute(0, 2, 3, 1).reshape(2, 30, 64)
    do, d_out, _ = M.linear_mxfp4_bwd(d, o_kept, seed=seeds[2:3])
    dq, dk, dv = C.cross_attention_bwd(do.view(2, 30, 2, 32), q, kv[:, :, 0], kv[:, :, 1], o, lse, key_mask=mask)
    _, d_q, _ = M.linear_mxfp4_bwd(dq.view(2, 30, 64), q_kept, seed=seeds[1:2])
    d_states, d_kv, _ = M.linear_mxfp4_bwd(torch.stack((dk, dv), 2).view(2, 11, 128), k_kept, seed=seeds[:1])
    for got, want in ((block.out.weight.grad, d_out), (block.q.weight.grad, d_q), (block.kv.weight.grad, d_kv),
                      (states.grad, d_states)):
        assert want.any() and torch.equal(got, want)
    assert x.grad.isfinite().all() and block.norm.weight.grad.any()


def test_prompt_kept_in_four_bits():
    g = torch.Generator().manual_seed(7)
    m = _model(text=_four()).eval()
    x, t, tokens = _images(4, g), torch.tensor([3, 10, 40, 90], device="cuda"), _tokens(4, 20, g)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        plain = m(x, t)
        m.keep_prompt(tokens)
        whole, seen = m._kept
        sixteen = m(x, t)
        m.keep_prompt(tokens, bits=4)
        four = m(x, t)
        assert not torch.equal(four, plain) and four.isfinite().all()
        for name, kv in m._kept[0].items():
            assert all(torch.equal(a, b) for a, b in zip(kv, M.quantize_mxfp4(whole[name])))
        assert not torch.equal(four, sixteen)
        m.keep_weights()
        assert torch.equal(m(x, t), four)
        m.keep_weights(False)
        m.keep_prompt(None)
        assert torch.equal(m(x, t), plain)
        m.keep_prompt(tokens, bits=4)
        assert torch.equal(m(x, t), four)
    with torch.autocast("cuda", dtype=torch.bfloat16), pytest.raises(ValueError, match="no gradient"):
        m(x, t)
    m.train().prompt = tokens       # training takes the prompt
    with torch.autocast("cuda", dtype=torch.bfloat16):
        m(x, t).float().square().mean().backward()
    assert m.text.weight.grad.any()


def test_a_prompt_of_sixteen_bit_projections_kept_in_four():
    g = torch.Generator().manual_seed(8)
    m = _model().eval()
    x, t, tokens = _images(3, g), torch.tensor([3, 10, 40], device="cuda"), _tokens(3, 12, g)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        m.keep_prompt(tokens, bits=4)
        y = m(x, t)
        m.keep_weights()            # (there are none to lay out)
        assert torch.equal(m(x, t), y) and y.isfinite().all()


def test_training_is_deterministic_and_reaches_every_parameter(seeds):
    g = torch.Generator().manual_seed(9)
    m = _model(text=_four(p_drop=0.1), p_drop=0.1).train()
    x, t, tokens = _images(4, g), torch.tensor([3, 10, 40, 90], device="cuda"), _tokens(4, 20, g)

    def grads():
        m.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            m(x, t, tokens).float().square().mean().backward()
        return {n: p.grad.clone() for n, p in m.named_parameters() if n.startswith(("cross.", "text."))}
    first, again = grads(), grads()
    for n, v in first.items():
        assert v.any() and v.isfinite().all() and torch.equal(again[n], v), n
    seeds.add_(1)
    other = grads()
    assert not torch.equal(other["cross.mid.q.weight"], first["cross.mid.q.weight"])


def test_captured_steps_are_the_eager_ones_to_the_bit(seeds):
    g = torch.Generator().manual_seed(11)
    data = [(_images(8, g), torch.randint(0, 100, (8,), generator=g).cuda(), _images(8, g), _tokens(8, 12, g))
            for _ in range(4)]

    def state():
        s = T.TrainState(_config(), 8, max_t=100, text=_four(), prompt_length=12, fixed_noise=True, ema_beta=0.9,
                         seed=1)
        s.set_batch(*data[0])
        return s

    def walk(s, step):
        losses = []
        for i in range(6):
            s.set_batch(*data[i % 4])
            seeds.copy_(torch.arange(1, 65, device="cuda") * 104729 + i)
            s.loss_acc.zero_()
            step()
            torch.cuda.synchronize()
            losses.append(float(s.loss_acc))
        return losses
    a, b = state(), state()
    a.capture(warmup=3)
    for _ in range(3):
        b.eager_step()
    assert walk(a, a.replay) == walk(b, b.eager_step)
    for (n, p), q in zip(a.model.named_parameters(), b.model.parameters()):
        assert torch.equal(p, q), n
    assert a.model.cross["mid"].q.weight.grad.any()


def test_operators_compile():
    g = torch.Generator().manual_seed(12)
    x = torch.randn((40, 96), generator=g).bfloat16().cuda()
    w = torch.randn((128, 96), generator=g).cuda()
    q = torch.randn((2, 9, 2, 32), generator=g).bfloat16().cuda()
    seed = torch.tensor([77], device="cuda")

    def f(x, w):
        return M.linear_mxfp4(x * 2, w, stochastic=True, seed=seed) * 3

    def serve(x, w):
        o = M.mxfp4_operand(w)
        y = M.linear_mxfp4_fwd(x * 2, o)
        kv = M.quantize_mxfp4(y[:32].reshape(2, 16, 2, 2, 32))
        return M.cross_attention_mxfp4(q * 2, kv) + M.dequantize_mxfp4(kv)[0, 0, 0]

    def run(fn):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = fn(a, b)
        y.float().square().sum().backward()
        return y.detach(), a.grad, b.grad
    want = run(f)
    with torch.no_grad():
        served = serve(x, w)
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        torch._dynamo.reset()
        fn = torch.compile(f, backend="aot_eager")
        for _ in range(2):
            assert all(torch.equal(a, b) for a, b in zip(run(fn), want))
        torch._dynamo.reset()
        fn = torch.compile(serve, backend="aot_eager")
        with torch.no_grad():
            for _ in range(2):
                assert torch.equal(fn(x, w), served)
    assert not [str(w.message) for w in seen if "dpa_fast_calls" in str(w.message) or "builtin" in str(w.message)]


def test_text_unet_compiles(seeds):
    m = _model(text=_four()).train()
    g = torch.Generator().manual_seed(13)
    x, t, tokens = _images(2, g), torch.tensor([3, 70], device="cuda"), _tokens(2, 12, g)

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
        assert all(torch.equal(a, b) for a, b in zip(step(fn), want))
    m.eval()
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        m.keep_prompt(tokens, bits=4)
        m.keep_weights()
        want = m(x, t)
        assert torch.equal(fn(x, t), want)


@pytest.mark.parametrize("length", [0, 1])
def test_shortest_prompts_kept_in_four_bits(length):
    g = torch.Generator().manual_seed(14)
    m = _model(text=_four()).eval()
    x, t = _images(2, g), torch.tensor([3, 70], device="cuda")
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        plain = m(x, t)
        m.keep_prompt(torch.zeros((2, length), dtype=torch.int64, device="cuda"), bits=4)
        assert torch.equal(m(x, t), plain)      # no token but the padding


def test_two_graphs_and_eager_calls_between():
    """Two captured graphs of split products and split keys, whose workspaces are their own, replayed in turn."""
    g = torch.Generator().manual_seed(15)
    w = M.mxfp4_operand(torch.randn((96, 8192), generator=g).bfloat16().cuda())
    kv = M.quantize_mxfp4(torch.randn((2, 4000, 2, 1, 64), generator=g).bfloat16().cuda())
    xs = [torch.zeros((100, 8192), device="cuda", dtype=torch.bfloat16) for _ in range(2)]

    def run(x):
        y = M.linear_mxfp4_fwd(x, w)
        return y, M.cross_attention_mxfp4(y[:, :64].reshape(2, 50, 1, 64)[:, :4], kv)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        run(xs[0])
    torch.cuda.current_stream().wait_stream(stream)
    graphs, outs = [], []
    for x in xs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(x))
    for i in range(4):
        for x in xs:
            x.copy_(torch.randn(x.shape, generator=g).bfloat16())
        graphs[i % 2].replay()
        want = [run(x) for x in xs]
        graphs[1 - i % 2].replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b)), i


def test_example_runs():
    spec = importlib.util.spec_from_file_location("text_to_image", os.path.join(ROOT, "examples", "text_to_image.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    losses = ex.main(["--steps", "60", "--batch", "16", "--max-t", "20", "--mxfp4", "--prompts", "red disc", ""])
    assert len(losses) == 2 and all(0 < x < float("inf") for x in losses)
