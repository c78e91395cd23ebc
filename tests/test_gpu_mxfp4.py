"""MXFP4 quantisation, operands, products and gradients against their definition in 64 bits. Codes, scales and
rounded values are exact; a product differs by its fp32 sums (K + 1 roundings of the sum of magnitudes at
most) and the rounding of the output, half a step."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import mxfp4_reference as R
from conftest import dpa_mod

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def M():
    return dpa_mod("mxfp4")


def randn(shape, seed, dtype, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * std
    # a few loud columns, and blocks of zeros
    x[..., ::37] *= 9.0
    if x.shape[-1] > 64:
        x[..., 32:64] = 0.0
    return x.to(dtype)


def seed_of(n: int) -> torch.Tensor:
    return torch.tensor([n], dtype=torch.int64, device="cuda")


def check_dense(M, x, what):
    print(f"quantize {what} {x.dtype} {tuple(x.shape)}", flush=True)
    q = M.quantize_mxfp4(x.cuda())
    code, byte = R.quantize(x)
    assert np.array_equal(q.scales.cpu().numpy(), byte), what
    got = R.unpack(q.data)
    there = code >= 0
    assert np.array_equal(got[there], code[there]), what
    want = R.values_of(code, byte)
    for dtype in (torch.bfloat16, torch.float32):
        y = M.dequantize_mxfp4(q, dtype).cpu().double()
        assert torch.equal(torch.nan_to_num(y, 1e300), torch.nan_to_num(want, 1e300)), (what, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(32,), (1, 64), (3, 5, 96), (77, 2, 4, 64), (1000, 1024), (0, 32)])
def test_quantize_is_exact(M, dtype, shape):
    check_dense(M, randn(shape, 1, dtype) if math.prod(shape) else torch.zeros(shape, dtype=dtype), "random")


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_borders_and_extremes(M, dtype):
    """Every midpoint and its neighbours at each power that the type has, the largest and smallest blocks, zeros of
    both signs, and blocks with an infinity or a NaN among ordinary ones."""
    mids = [0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0]
    near = torch.tensor([s * m * (1 + d) for m in mids for d in (0.0, 2.0**-7, -(2.0**-8)) for s in (1, -1)])
    rows = []
    info = torch.finfo(dtype)
    low, high = math.frexp(info.smallest_normal)[1], math.frexp(info.max)[1] - 4
    for k in range(low, high + 1, 1 if dtype == torch.float16 else 9):
        block = torch.ldexp(near, torch.tensor(float(k)))
        rows += [block[:32], block[32:64], block[64:96]]
    rows += [torch.zeros(32), -torch.zeros(32), torch.full((32,), info.max), torch.full((32,), -info.tiny)]
    for bad in (math.inf, -math.inf, math.nan):
        r = torch.arange(32.0)
        r[17] = bad
        rows += [r, torch.arange(32.0)]
    tiny = torch.zeros(32)
    tiny[3], tiny[4] = info.smallest_normal / 4, -info.smallest_normal / 2      # subnormal
    rows.append(tiny)
    check_dense(M, torch.stack(rows).to(dtype), "borders")


def test_dequantize_every_code_and_scale(M):
    code = np.tile(np.arange(16), 2)[None].repeat(256, 0)
    byte = np.arange(256)[:, None]
    want = R.values_of(code, byte)
    q = M.MXFP4(R.pack(code).cuda(), torch.from_numpy(byte.astype(np.uint8)).cuda())
    for dtype in DTYPES:
        y = M.dequantize_mxfp4(q, dtype).cpu()
        ref = want.to(dtype)
        assert torch.equal(torch.isnan(y), torch.isnan(ref))
        assert torch.equal(torch.nan_to_num(y, 7.0), torch.nan_to_num(ref, 7.0)), dtype
        if dtype != torch.float16:      # exact up to byte 252 (6 2^125 < 2^128; of 253, 4 2^126 is 2^128)
            assert torch.equal(ref.double()[:253], want[:253])


def test_quantize_copies_what_it_does_not_read_in_place(M):
    x = randn((64, 96), 3, torch.bfloat16).cuda()
    want = M.quantize_mxfp4(x.t()[:, :32].contiguous())
    got = M.quantize_mxfp4(x.t()[:, :32])
    assert torch.equal(got.data, want.data) and torch.equal(got.scales, want.scales)
    flat = torch.randn(32 * 9 + 1, device="cuda")[1:].view(9, 32)           # 4 B off
    want = M.quantize_mxfp4(flat.clone())
    got = M.quantize_mxfp4(flat)
    assert torch.equal(got.data, want.data)
    y = M.dequantize_mxfp4(M.MXFP4(got.data[2:], got.scales[2:]))
    assert torch.equal(y, M.dequantize_mxfp4(got)[2:])


# ---- operands: the product with an identity gives them back ---------------------------------
def operand_values(M, o):
    eye = M.mxfp4_operand(torch.eye(o.cols, device="cuda", dtype=torch.bfloat16))
    return M._product(o, eye, None, torch.float32).cpu().double()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (5, 33), (32, 256), (77, 100), (130, 260), (300, 513), (515, 128),
                                   (1030, 70)])
@pytest.mark.parametrize("seed", [None, 1234567])
def test_operands_hold_the_rounded_values(M, dtype, shape, seed):
    x = randn(shape, 5, dtype)
    s = None if seed is None else seed_of(seed)
    rows, cols = M.mxfp4_operands(x.cuda(), seed=s)
    want_r, want_c = R.rounded(x, -1, seed), R.rounded(x, 0, seed)
    assert torch.equal(operand_values(M, rows), want_r)
    assert torch.equal(operand_values(M, cols), want_c.t())
    alone = M.mxfp4_operand(x.cuda(), seed=s)
    assert torch.equal(operand_values(M, alone), want_r)
    # rows further apart, and columns that are not dense (a copy)
    wide = torch.full((shape[0], shape[1] + 3), math.nan, dtype=dtype, device="cuda")
    wide[:, 1:1 + shape[1]] = x.cuda()
    r2, c2 = M.mxfp4_operands(wide[:, 1:1 + shape[1]], seed=s)
    assert torch.equal(operand_values(M, r2), want_r) and torch.equal(operand_values(M, c2), want_c.t())
    t = M.mxfp4_operand(x.cuda().t().contiguous().t(), seed=s)
    assert torch.equal(operand_values(M, t), want_r)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_operands_take_the_wide_form(M, dtype):
    """The bytes of the transpose the other way round, and of some of the rows alone."""
    def panels(o):
        return o.data[:-(-o.rows // 16) * 16 * -(-o.cols // 256) * 128].view(-1, -(-o.rows // 16) * 16, 64)[:, :o.rows]
    x = randn((16384, 2100), 6, dtype).cuda()
    n, k = x.shape
    rows, cols = M.mxfp4_operands(x)
    t_rows, t_cols = M.mxfp4_operands(x.t().contiguous())
    assert torch.equal(panels(rows), panels(t_cols)) and torch.equal(panels(cols), panels(t_rows))
    y = M.mxfp4_operand(randn((40, n), 8, dtype).cuda())
    assert torch.equal(M._product(cols, y, None, torch.float32), M._product(t_rows, y, None, torch.float32))
    pick = torch.tensor([0, 31, 257, 4000, 16383], device="cuda")
    small = M.mxfp4_operand(x[pick].contiguous())
    y = M.mxfp4_operand(randn((40, k), 7, dtype).cuda())
    assert torch.equal(M._product(small, y, None, torch.float32), M._product(rows, y, None, torch.float32)[pick])
    s = seed_of(77)
    r1, c1 = M.mxfp4_operands(x, seed=s)
    r2 = M.mxfp4_operand(x, seed=s)
    assert torch.equal(panels(r1), panels(r2))
    few = M.mxfp4_operands(x[:300], seed=s)
    assert torch.equal(operand_values(M, few[1]), R.rounded(x[:300].cpu(), 0, 77).t())
    assert torch.equal(panels(c1)[:2], panels(few[1])[:2])


def test_stochastic_rounding_keeps_the_mean(M):
    """1024 draws of every element: a mean of n draws between two neighbours a step apart strays by more than
    step / 2 sqrt(2 ln(2 / p) / n) (Hoeffding) with probability p; p = 1e-9 over 512 elements."""
    x = torch.linspace(-7.9, 7.9, 512).view(1, -1)
    n = 1024
    seeds = torch.arange(n) * 7919 + 5
    total = torch.zeros(512, dtype=torch.float64)
    for s in seeds[:4].tolist():        # the kernel, then its definition, which it equals
        got = operand_values(M, M.mxfp4_operand(x.cuda(), seed=seed_of(s)))
        assert torch.equal(got, R.rounded(x, -1, s))
    for s in seeds.tolist():
        total += R.rounded(x, -1, s)[0]
    scale = R.quantize(x, R.random_bits(1, 512, 1))[1].astype(float)
    step = torch.from_numpy(2.0 * np.exp2(scale - 127)).repeat_interleave(32, 1)[0]
    assert (total / n - x[0].double()).abs().le(step * math.sqrt(2 * math.log(2e9) / n) / 2).all()


# ---- products ------------------------------------------------------------------------------
def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check_product(y, a, b, bias, dtype, what):
    """y against a b^T + bias in 64 bits: fp32 sums (each of K + 2 steps rounds to within 2^-24 of the sum of
    magnitudes; the matrix unit may truncate, a whole step) and the output's half step."""
    want = a @ b.t()
    size = a.abs() @ b.abs().t()
    if bias is not None:
        want = want + bias.double().cpu()
        size = size + bias.double().abs().cpu()
    sums = (a.shape[1] + 2) * 2.0**-23 * size
    err = (y.cpu().double() - want).abs()
    bound = sums + half_step(dtype) * (want.abs() + sums) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert (err <= bound).all(), (what, float((err - bound).max()), float(err.max()))


SIZES = [(1, 1, 1), (1, 512, 2048), (1, 8192, 96), (2, 33, 17), (15, 257, 40), (16, 5120, 130), (17, 300, 64), (33, 4096, 65),
         (64, 700, 200), (65, 256, 128), (100, 1000, 99), (128, 96, 128), (129, 520, 257), (200, 4100, 130),
         (1031, 1000, 1023), (300, 31, 515), (70, 9000, 16), (2500, 64, 9)]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_forward(M, m, k, n, dtype):
    x, w = randn((m, k), 7, dtype), randn((n, k), 8, dtype, 1 / math.sqrt(k))
    bias = randn((n,), 9, torch.float32) if (m + n) % 2 else None
    xd, wd, bd = x.cuda(), w.cuda(), None if bias is None else bias.cuda()
    a, b = R.rounded(x), R.rounded(w)
    y = M.linear_mxfp4_fwd(xd, wd, bd)
    assert y.dtype == dtype and y.shape == (m, n)
    check_product(y, a, b, bias, dtype, "weight")
    kept = M.mxfp4_operand(wd)
    assert torch.equal(M.linear_mxfp4_fwd(xd, kept, bd), y)
    for other in DTYPES:
        if other != dtype:
            check_product(M.linear_mxfp4_fwd(xd, kept, bd, out_dtype=other), a, b, bias, other, "out_dtype")


def test_linear_many_columns_and_rows(M):
    """Tiles of every kind in one product, checked by rows and columns picked from it."""
    m, k, n = 4100, 1536, 2050
    x, w = randn((m, k), 11, torch.bfloat16), randn((n, k), 12, torch.bfloat16, 0.03)
    y = M.linear_mxfp4_fwd(x.cuda(), w.cuda(), out_dtype=torch.float32).cpu()
    a, b = R.rounded(x), R.rounded(w)
    pick = torch.tensor([0, 1, 127, 128, 255, 1000, 4095, 4096, 4099])
    check_product(y[pick], a[pick], b, None, torch.float32, "rows")
    pick = torch.tensor([0, 3, 16, 63, 64, 129, 1023, 2047, 2048, 2049])
    check_product(y[:, pick], a, b[pick], None, torch.float32, "columns")


def test_linear_carries_nan_of_a_block_to_its_rows_and_columns_only(M):
    x, w = randn((130, 200), 13, torch.bfloat16), randn((70, 200), 14, torch.bfloat16)
    x[7, 40] = math.inf
    w[69, 199] = math.nan
    for rows in (slice(0, 130), slice(0, 10)):
        y = M.linear_mxfp4_fwd(x[rows].cuda(), w.cuda(), out_dtype=torch.float32).cpu()
        assert torch.isnan(y[7]).all() and torch.isnan(y[:, 69]).all()
        there = torch.ones_like(y, dtype=torch.bool)
        there[7], there[:, 69] = False, False
        assert torch.isfinite(y[there]).all()


def test_linear_takes_any_leading_shape_and_strides(M):
    x, w = randn((3, 5, 160), 15, torch.bfloat16).cuda(), randn((40, 160), 16, torch.float32).cuda()
    y = M.linear_mxfp4_fwd(x, w)
    assert y.shape == (3, 5, 40)
    assert torch.equal(M.linear_mxfp4_fwd(x.transpose(0, 1), w), y.transpose(0, 1))
    assert torch.equal(M.linear_mxfp4_fwd(x[1, 2], w), y[1, 2])
    assert M.linear_mxfp4_fwd(x[:0], w).shape == (0, 5, 40)
    wide = torch.full((15, 200), math.nan, device="cuda", dtype=torch.bfloat16)
    wide[:, 8:168] = x.view(15, 160)
    assert torch.equal(M.linear_mxfp4_fwd(wide[:, 8:168], w), y.view(15, 40))
    assert torch.equal(M.linear_mxfp4_fwd(x, w.t().contiguous().t()), y)


# ---- gradients -----------------------------------------------------------------------------
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (3, 40, 33), (65, 129, 70), (128, 256, 128), (1000, 96, 257), (3850, 65, 130),
                                   (40, 700, 1500)])
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                          (torch.float32, torch.float32)])
@pytest.mark.parametrize("seed", [None, 99])
def test_linear_gradients_are_the_formulas(M, m, k, n, dtype, wdtype, seed):
    x, w, dy = randn((m, k), 17, dtype), randn((n, k), 18, wdtype), randn((m, n), 19, dtype, 0.1)
    bias = randn((n,), 20, torch.float32)
    y, kept = M.linear_mxfp4_train_fwd(x.cuda(), w.cuda(), bias.cuda())
    assert torch.equal(y, M.linear_mxfp4_fwd(x.cuda(), w.cuda(), bias.cuda()))
    s = None if seed is None else seed_of(seed)
    dx, dw, db = M.linear_mxfp4_bwd(dy.cuda(), kept, seed=s)
    assert dx.dtype == dtype and dw.dtype == wdtype and db.dtype == torch.float32
    check_product(dx, R.rounded(dy, -1, seed), R.rounded(w, 0).t().contiguous(), None, dtype, "dx")
    check_product(dw, R.rounded(dy, 0, seed).t().contiguous(), R.rounded(x, 0).t().contiguous(), None, wdtype, "dw")
    err = (db.cpu().double() - dy.double().sum(0)).abs()
    assert (err <= m * 2.0**-24 * dy.double().abs().sum(0)).all()
    again = M.linear_mxfp4_bwd(dy.cuda(), kept, seed=s)
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))


def on_grid(shape, seed):
    """Small whole numbers, a 6 in every block of every direction: MXFP4 holds them as they are."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-3, 4, shape, generator=g).float()
    x[::32], x[:, ::32] = 6.0, 6.0
    return x


def test_linear_gradients_are_the_differences(M):
    """On numbers that the roundings keep, the loss sum(y dy) is linear in x and in w: moving one element by 1
    changes it by exactly the gradient."""
    m, k, n = 70, 96, 64
    x, w, dy = on_grid((m, k), 21).cuda(), on_grid((n, k), 22).cuda(), on_grid((m, n), 23).cuda()
    x[5, 7], w[9, 11] = 1.0, 2.0
    _, kept = M.linear_mxfp4_train_fwd(x, w)
    dx, dw, db = M.linear_mxfp4_bwd(dy, kept)
    assert db is None

    def loss(x, w):
        return (M.linear_mxfp4_fwd(x, w).double() * dy.double()).sum()
    at = loss(x, w)
    x2, w2 = x.clone(), w.clone()
    x2[5, 7] += 1.0
    w2[9, 11] += 1.0
    assert loss(x2, w) - at == dx[5, 7].double()
    assert loss(x, w2) - at == dw[9, 11].double()


@pytest.mark.parametrize("need", ["x", "w", "b", "xw", "xwb"])
def test_linear_autograd(M, need):
    """Only the gradients that are asked for, in the parameters' dtypes, equal to the op-level ones."""
    x = randn((4, 30, 130), 24, torch.bfloat16).cuda().requires_grad_("x" in need)
    w = randn((70, 130), 25, torch.float32).cuda().requires_grad_("w" in need)
    b = randn((70,), 26, torch.bfloat16).cuda().requires_grad_("b" in need)
    dy = randn((4, 30, 70), 27, torch.bfloat16).cuda()
    y = M.linear_mxfp4(x, w, b, stochastic=True, seed=seed_of(5))
    y.backward(dy)
    ref, kept = M.linear_mxfp4_train_fwd(x.detach(), w.detach(), b.detach())
    dx, dw, db = M.linear_mxfp4_bwd(dy, kept, seed=seed_of(5))
    assert torch.equal(y, ref)
    for t, g, name in ((x, dx, "x"), (w, dw, "w"), (b, db, "b")):
        if name in need:
            assert t.grad.dtype == t.dtype and torch.equal(t.grad, g.to(t.dtype))
        else:
            assert t.grad is None
    # a broadcast gradient (strides of 0), and a weight that two calls share
    if need == "xwb":
        for t in (x, w, b):
            t.grad = None
        (M.linear_mxfp4(x, w, b).sum() + M.linear_mxfp4(x, w).sum()).backward()
        ones = torch.ones_like(dy)
        dx, dw, db = M.linear_mxfp4_bwd(ones, kept)
        assert torch.equal(x.grad, dx + dx) and torch.equal(w.grad, dw + dw) and torch.equal(b.grad, db.to(b.dtype))


def test_linear_autocast_and_module(M):
    x = randn((6, 96), 28, torch.float32).cuda()
    layer = M.LinearMXFP4(96, 40).cuda()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layer(x)
        z = layer(x.to(torch.bfloat16))
    assert y.dtype == z.dtype == torch.bfloat16
    assert torch.equal(y, M.linear_mxfp4_fwd(x, layer.weight, layer.bias, out_dtype=torch.bfloat16))
    y.float().sum().backward()
    assert layer.weight.grad.dtype == torch.float32 and layer.bias.grad.shape == (40,)
    before = layer(x).detach()
    layer.keep_weight()
    with torch.no_grad():
        assert torch.equal(layer(x), before)
        layer.weight.mul_(2.0)
        assert torch.equal(layer(x), before)            # as it was
        layer.keep_weight(False)
        assert not torch.equal(layer(x), before)
    assert list(layer.state_dict()) == ["weight", "bias"]
    with pytest.raises(ValueError, match="gradients need the weight"):
        M.linear_mxfp4(x.requires_grad_(), M.mxfp4_operand(layer.weight.detach()))


def test_linear_in_a_captured_step(M):
    """Forward and backward in one graph, replayed with new inputs and eager work between, equal to eager."""
    x, dy = torch.zeros(200, 300, device="cuda", dtype=torch.bfloat16), torch.zeros(200, 90, device="cuda", dtype=torch.bfloat16)
    w, bias, seed = randn((90, 300), 29, torch.float32).cuda(), randn((90,), 30, torch.float32).cuda(), seed_of(3)

    def step():
        y, kept = M.linear_mxfp4_train_fwd(x, w, bias)
        return (y, *M.linear_mxfp4_bwd(dy, kept, seed=seed))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(randn((200, 300), 40 + i, torch.bfloat16))
        dy.copy_(randn((200, 90), 50 + i, torch.bfloat16))
        seed.fill_(1000 + i)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_calls_on_two_streams_do_not_meet(M):
    """Split products (with a workspace) on two streams at once."""
    x, w = randn((100, 8192), 31, torch.bfloat16).cuda(), randn((64, 8192), 32, torch.bfloat16).cuda()
    want = M.linear_mxfp4_fwd(x, w)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    torch.cuda.synchronize()
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(M.linear_mxfp4_fwd(x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_tensors_on_another_device_than_the_current_one(M, monkeypatch):
    """Their device is the current one for each launch (shown with the question for the current device turned)."""
    x, w = randn((70, 96), 61, torch.bfloat16).cuda(), randn((40, 96), 62, torch.bfloat16).cuda()
    want = M.linear_mxfp4_fwd(x, w)
    q4 = M.quantize_mxfp4(x)
    entered = []

    class On(torch.cuda.device):
        def __enter__(self):
            entered.append(self.idx)
            return super().__enter__()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 7)
    monkeypatch.setattr(torch.cuda, "device", On)
    assert torch.equal(M.linear_mxfp4_fwd(x, w), want) and entered == [0, 0]
    kept = M.mxfp4_operand(w)
    assert entered == [0, 0, 0]
    monkeypatch.undo()
    assert torch.equal(M.linear_mxfp4_fwd(x, kept), want)
    assert torch.equal(M.quantize_mxfp4(x).data, q4.data)
