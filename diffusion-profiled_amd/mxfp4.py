"""Microscaled 4-bit floating point (MXFP4) on the HIP library's kernels (``dpa_mxfp4_*``,
``dpa_cross_attention_mxfp4``): quantisation and back, the linear layer on 4-bit operands, and cross
attention over keys and values held in 4 bits. The reference quantises to e4m3 with one scale a tensor
(diffusion/fp8_kernels.py:518-601) and has no counterpart.

32 neighbours share a power of two: of largest magnitude amax they get 2^k, k = floor(log2 amax) - 2 and at
least -127, kept as the byte k + 127, and become e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives)
times it, to nearest even, what passes 6 as 6. A block with a NaN or an infinity gets the byte 255 and is
NaN throughout. Stochastic rounding (gradients) goes up or down so that the mean of a rounded element
is the element, by 16 bits of the counter hash of ``conditioning`` each; its k is one higher where amax would
pass 6, so that nothing is cut off.

Two arrangements: ``MXFP4``, a tensor in order, and ``MXFP4Operand``, a matrix as the product reads it.
As in ``conditioning``, each operator comes as functions of one launch sequence per direction (``*_fwd``,
``*_bwd``, which record nothing) and as a differentiable function. GPU tensors only; there is no fallback.
"""
from __future__ import annotations

import struct
from typing import Any, NamedTuple

import torch
import torch.nn as nn
from torch.amp.autocast_mode import custom_bwd, custom_fwd
from torch.autograd import forward_ad

from . import _lib
from .conditioning import (_DT, _between_graphs, _check_masks, _check_seed, _fast, _on_one_gpu, _ptr, _rows,
                           _scale_of, _strides, _workspace)
from .eager import apply
from .gn_silu import DROPOUT_SEEDS

BLOCK = 32
# DpaCrossAttentionMxfp4 of include/dpa_fp8.h: 9 pointers, the mask's stride, 5 x 3 strides, 7 sizes, the scale
_DESC = struct.Struct("=9Qq15q7if")


class MXFP4(NamedTuple):
    """A tensor [..., C], C a multiple of 32."""
    data: torch.Tensor      # uint8 [..., C / 2], the first of two elements in the low half
    scales: torch.Tensor    # uint8 [..., C / 32]

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.data.shape[:-1], 2 * self.data.shape[-1]))


class MXFP4Operand(NamedTuple):
    """A matrix [rows, cols] for a product that sums over its cols: any sizes, blocks along the rows, laid
    out by ``mxfp4_operand`` (include/dpa_fp8.h has the sizes; the order is the kernels')."""
    data: torch.Tensor
    rows: int
    cols: int


def _check_dtype(what: str, *dtypes: torch.dtype) -> None:
    for dt in dtypes:
        if dt not in _DT:
            raise ValueError(f"{what}: bf16, fp16 or fp32, got {dt}")


def _call(entry: str, *args) -> None:
    """An entry of the library on the current stream of the last argument's device, which is the current one for the
    launch."""
    *args, on = args
    if on.get_device() == torch.cuda.current_device():
        _lib.call(entry, *args, _lib.current_stream(on))
    else:
        with torch.cuda.device(on.device):
            _lib.call(entry, *args, _lib.current_stream(on))


def _has_tangent(*tensors: torch.Tensor | None) -> bool:
    """Whether one of them is a dual tensor of forward-mode differentiation (with gradients off too)."""
    if getattr(forward_ad, "_current_level", 0) < 0:
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


# ---- quantisation ------------------------------------------------------------------------
def quantize_mxfp4(x: torch.Tensor) -> MXFP4:
    """x [..., C] (bf16, fp16 or fp32; C a multiple of 32) in MXFP4, blocks along the last dimension."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(quantize_mxfp4, x)
    done = _fast().mxfp4_quantize(x)
    if done is not None:
        return MXFP4(*done)
    _check_dtype("quantize_mxfp4", x.dtype)
    if x.ndim < 1 or x.shape[-1] == 0 or x.shape[-1] % BLOCK:
        raise ValueError(f"quantize_mxfp4: the last dimension is a multiple of {BLOCK}, got {tuple(x.shape)}")
    _on_one_gpu(x)
    x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone()
    lead, c = x.shape[:-1], x.shape[-1]
    data = torch.empty((*lead, c // 2), device=x.device, dtype=torch.uint8)
    scales = torch.empty((*lead, c // BLOCK), device=x.device, dtype=torch.uint8)
    _call("dpa_mxfp4_quantize", x.data_ptr(), _DT[x.dtype], x.numel(), data.data_ptr(), scales.data_ptr(),
              x)
    return MXFP4(data, scales)


def _check_mxfp4(q: MXFP4, what: str) -> None:
    if q.data.dtype != torch.uint8 or q.scales.dtype != torch.uint8:
        raise ValueError(f"{what}: data and scales are uint8, got {q.data.dtype} and {q.scales.dtype}")
    if q.data.ndim < 1 or q.data.shape[:-1] != q.scales.shape[:-1] or q.data.shape[-1] != 16 * q.scales.shape[-1]:
        raise ValueError(f"{what}: data {tuple(q.data.shape)} and scales {tuple(q.scales.shape)} do not go "
                         "together (16 bytes of data to a scale)")
    _on_one_gpu(q.data, q.scales)


def dequantize_mxfp4(q: MXFP4, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of q in dtype: exact in bf16 and fp32, rounded once in fp16."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(dequantize_mxfp4, q, dtype)
    y = _fast().mxfp4_dequantize(q.data, q.scales, dtype)
    if y is not None:
        return y
    _check_dtype("dequantize_mxfp4", dtype)
    _check_mxfp4(q, "dequantize_mxfp4")
    data, scales = q.data.contiguous(), q.scales.contiguous()
    if data.data_ptr() % 4:
        data = data.clone()
    y = torch.empty(q.shape, device=data.device, dtype=dtype)
    _call("dpa_mxfp4_dequantize", data.data_ptr(), scales.data_ptr(), y.data_ptr(), _DT[dtype], y.numel(),
              data)
    return y


# ---- operands ----------------------------------------------------------------------------
def _new_operand(rows: int, cols: int, device) -> MXFP4Operand:
    nbytes = _lib.query("dpa_mxfp4_operand_bytes", rows, cols)
    if nbytes == 0 and rows and cols:
        raise ValueError(f"mxfp4 operand: {rows} x {cols} is beyond what the kernels take")
    return MXFP4Operand(torch.empty(nbytes, device=device, dtype=torch.uint8), rows, cols)


def _matrix(x: torch.Tensor) -> torch.Tensor:
    """x as rows of dense columns."""
    return x if x.stride(1) == 1 and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()


def _operands(x: torch.Tensor, rows: bool, cols: bool, seed: torch.Tensor | None, sums: torch.Tensor | None = None):
    """x's operand, that of its transpose, or both; with the latter the sums down the columns of every 64 rows."""
    _check_dtype("mxfp4 operand", x.dtype)
    if x.ndim != 2 or x.shape[1] == 0:
        raise ValueError(f"mxfp4 operand: a matrix of at least one column, got {tuple(x.shape)}")
    _on_one_gpu(x)
    if seed is not None:
        _check_seed(seed, x, "mxfp4 operand")
    x = _matrix(x)
    m, k = x.shape
    r = _new_operand(m, k, x.device) if rows else None
    c = _new_operand(k, m, x.device) if cols else None
    if m:
        _call("dpa_mxfp4_operands", x.data_ptr(), _DT[x.dtype], m, k, x.stride(0) if m > 1 else k,
                  _ptr(r and r.data), _ptr(c and c.data), _ptr(sums), _ptr(seed), x)
    return r, c


def mxfp4_operand(x: torch.Tensor, *, seed: torch.Tensor | None = None) -> MXFP4Operand:
    """x [rows, cols] (bf16, fp16 or fp32) as an operand of ``linear_mxfp4_fwd``: a weight laid out once, for
    instance. seed: an int64 tensor of one element on the device, for stochastic rounding."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(mxfp4_operand, x, seed=seed)
    return _operands(x, True, False, seed)[0]


def mxfp4_operands(x: torch.Tensor, *, seed: torch.Tensor | None = None) -> tuple[MXFP4Operand, MXFP4Operand]:
    """The operands of x and of its transpose (blocks down the columns of x), from one read of it."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(mxfp4_operands, x, seed=seed)
    return _operands(x, True, True, seed)


def _product(a: MXFP4Operand, b: MXFP4Operand, bias: torch.Tensor | None, dtype: torch.dtype) -> torch.Tensor:
    """a b^T (+ bias)"""
    m, n, k = a.rows, b.rows, a.cols
    y = torch.empty((m, n), device=a.data.device, dtype=dtype)
    if m and n:
        nbytes = _lib.query("dpa_mxfp4_gemm_workspace_bytes", m, n, k)
        ws = _workspace(nbytes, a.data.device)
        _call("dpa_mxfp4_gemm", a.data.data_ptr(), b.data.data_ptr(), _ptr(bias), y.data_ptr(), _DT[dtype], m, n, k,
                  _ptr(ws), nbytes, a.data)
    return y


# ---- the linear layer --------------------------------------------------------------------
def _check_operand(w: MXFP4Operand) -> None:
    if (w.data.dtype != torch.uint8 or not w.data.is_contiguous() or w.data.data_ptr() % 16
            or w.data.numel() != _lib.query("dpa_mxfp4_operand_bytes", w.rows, w.cols)):
        raise ValueError(f"linear_mxfp4: not an operand of {w.rows} x {w.cols}: {w.data.dtype} {tuple(w.data.shape)}")
    _on_one_gpu(w.data)


def _check_linear(x: torch.Tensor, n: int, k: int, bias: torch.Tensor | None, out_dtype: torch.dtype | None):
    """(x as a matrix, bias in fp32, the output's dtype)"""
    out_dtype = x.dtype if out_dtype is None else out_dtype
    _check_dtype("linear_mxfp4", x.dtype, out_dtype)
    if x.ndim < 1 or x.shape[-1] != k or k == 0:
        raise ValueError(f"linear_mxfp4: x {tuple(x.shape)} does not go with a weight [{n}, {k}]")
    if bias is not None:
        if bias.shape != (n,):
            raise ValueError(f"linear_mxfp4: bias {tuple(bias.shape)} does not go with a weight [{n}, {k}]")
        _check_dtype("linear_mxfp4", bias.dtype)
        _on_one_gpu(x, bias)
        bias = bias.float().contiguous()
    return x.reshape(-1, k), bias, out_dtype


def linear_mxfp4_fwd(x: torch.Tensor, weight: torch.Tensor | MXFP4Operand, bias: torch.Tensor | None = None, *,
                     out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Q(x) Q(weight)^T + bias in out_dtype (x's by default): x [..., K] and weight [N, K] rounded to MXFP4 with
    blocks along K, sums and bias in fp32, one rounding. weight: bf16, fp16 or fp32, or an operand made of it
    before (``mxfp4_operand``). The last block of a row may be shorter. Sizes: a matrix of r rows and c columns has
    (r rounded up to 16) * ceil(c / 512) below 2^25, and the same with r and c exchanged; K is at most 2^24 and the output
    has less than 2^33 elements."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(linear_mxfp4_fwd, x, weight, bias, out_dtype=out_dtype)
    if isinstance(weight, MXFP4Operand):
        y = _fast().mxfp4_linear(x, weight.data, weight.rows, weight.cols, bias, out_dtype)
        if y is not None:
            return y
        _check_operand(weight)
        _on_one_gpu(x, weight.data)
        n, k = weight.rows, weight.cols
    else:
        if weight.ndim != 2:
            raise ValueError(f"linear_mxfp4: the weight is [N, K], got {tuple(weight.shape)}")
        _on_one_gpu(x, weight)
        n, k = weight.shape
    x2, b32, dtype = _check_linear(x, n, k, bias, out_dtype)
    w = weight if isinstance(weight, MXFP4Operand) else _operands(weight, True, False, None)[0]
    x2 = _matrix(x2)
    m = x2.shape[0]
    y = torch.empty((m, n), device=x.device, dtype=dtype)
    if m and n:
        _new_operand(m, k, "meta")      # (refuses sizes beyond the kernels')
        ld = x2.stride(0) if m > 1 else k
        nbytes = _lib.query("dpa_mxfp4_linear_workspace_bytes", x2.data_ptr(), _DT[x2.dtype], ld, m, n, k)
        ws = _workspace(nbytes, x.device)
        _call("dpa_mxfp4_linear", x2.data_ptr(), _DT[x2.dtype], ld, w.data.data_ptr(), _ptr(b32), y.data_ptr(),
                  _DT[dtype], m, n, k, _ptr(ws), nbytes, x2)
    return y.view(*x.shape[:-1], n)


class LinearKept(NamedTuple):
    """What the gradients need of a forward: the operands of the transposes of x and of the weight (None where
    its product is not wanted)."""
    x: MXFP4Operand | None
    weight: MXFP4Operand | None
    shape: torch.Size       # of x
    out_features: int
    dtype: torch.dtype      # of x, and so of its gradient
    weight_dtype: torch.dtype
    bias: bool


def _check_products(m: int, n: int, k: int, want_dx: bool, want_dw: bool) -> None:
    """Refuses, before anything is launched, sizes of which one of a training step's products is beyond the kernels."""
    if m == 0 or n == 0:
        return
    for what, size in (("output", (m, n, k)), ("dx", (m, k, n) if want_dx else None), ("dweight", (n, k, m) if want_dw else None)):
        if size and _lib.query("dpa_mxfp4_gemm_plan", *size, 0, None):
            raise ValueError(f"linear_mxfp4: {m} rows of {k} with a weight [{n}, {k}]: the product of {what}, {size[0]} x {size[1]} "
                             f"over {size[2]}, is beyond what the kernels take")


def _train_fwd(x, weight, bias, out_dtype, want_dx: bool, want_dw: bool):
    if weight.ndim != 2:
        raise ValueError(f"linear_mxfp4: the weight is [N, K], got {tuple(weight.shape)}")
    _on_one_gpu(x, weight)
    n, k = weight.shape
    x2, b32, dtype = _check_linear(x, n, k, bias, out_dtype)
    _check_products(x2.shape[0], n, k, want_dx, want_dw)
    xr, xc = _operands(x2, True, want_dw, None)
    wr, wc = _operands(weight, True, want_dx, None)
    y = _product(xr, wr, b32, dtype).view(*x.shape[:-1], n)
    return y, LinearKept(xc, wc, x.shape, n, x.dtype, weight.dtype, bias is not None)


def linear_mxfp4_train_fwd(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                           out_dtype: torch.dtype | None = None) -> tuple[torch.Tensor, LinearKept]:
    """``linear_mxfp4_fwd``, and what ``linear_mxfp4_bwd`` needs of it (17/32 byte an element of x and of
    the weight). Sizes whose gradients are products beyond the kernels (more than 2^24 rows of x or of the weight) are
    refused here."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(linear_mxfp4_train_fwd, x, weight, bias, out_dtype=out_dtype)
    done = _fast().mxfp4_train_fwd(x, weight, bias, out_dtype)
    if done is not None:
        (y, xc, wc), (n, k) = done, weight.shape
        return y, LinearKept(MXFP4Operand(xc, k, x.numel() // k), MXFP4Operand(wc, k, n), x.shape, n, x.dtype,
                             weight.dtype, bias is not None)
    return _train_fwd(x, weight, bias, out_dtype, True, True)


def _column_sum(x: torch.Tensor) -> torch.Tensor:
    m, n = x.shape
    y = torch.empty(n, device=x.device, dtype=torch.float32)
    nbytes = _lib.query("dpa_column_sum_workspace_bytes", m, n)
    ws = _workspace(nbytes, x.device)
    _call("dpa_column_sum", x.data_ptr(), _DT[x.dtype], m, n, x.stride(0) if m > 1 else n, y.data_ptr(), _ptr(ws),
              nbytes, x)
    return y


def linear_mxfp4_bwd(dy: torch.Tensor, kept: LinearKept, *, seed: torch.Tensor | None = None
                     ) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """(dx, dweight, dbias) from the output's gradient: dx = Q(dy) Q(weight), dweight = Q(dy)^T Q(x), each factor
    rounded to MXFP4 with blocks along the dimension that its product sums over, dx in x's dtype, dweight in
    the weight's, dbias (None without a bias) the sum of dy in fp32. seed: dy is rounded stochastically (int64
    tensor of one element on the device), else to nearest. Deterministic."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(linear_mxfp4_bwd, dy, kept, seed=seed)
    n, k = kept.out_features, kept.shape[-1]
    if kept.x is not None and kept.weight is not None and dy.shape[:-1] == kept.shape[:-1]:
        done = _fast().mxfp4_bwd(dy, kept.x.data, kept.weight.data, n, k, kept.dtype, kept.weight_dtype, kept.bias, seed)
        if done is not None:
            return done
    _check_dtype("linear_mxfp4", dy.dtype)
    if dy.shape != (*kept.shape[:-1], n):
        raise ValueError(f"linear_mxfp4: dy {tuple(dy.shape)} is not the output's {(*kept.shape[:-1], n)}")
    device = dy.device
    if dy.numel() == 0:
        dx = torch.zeros(kept.shape, device=device, dtype=kept.dtype) if kept.weight is not None else None
        dw = torch.zeros((n, k), device=device, dtype=kept.weight_dtype) if kept.x is not None else None
        return dx, dw, torch.zeros(n, device=device, dtype=torch.float32) if kept.bias else None
    for o in (kept.x, kept.weight):
        if o is not None:
            _check_operand(o)
            _on_one_gpu(dy, o.data)
    dy2 = _matrix(dy.reshape(-1, n))
    dx = dw = None
    summed = dy2
    if kept.weight is not None or kept.x is not None:
        part = None
        if kept.bias and kept.x is not None:
            part = summed = torch.empty((-(-dy2.shape[0] // 64), n), device=device, dtype=torch.float32)
        dyr, dyc = _operands(dy2, kept.weight is not None, kept.x is not None, seed, part)
        if kept.weight is not None:
            dx = _product(dyr, kept.weight, None, kept.dtype).view(kept.shape)
        if kept.x is not None:
            dw = _product(dyc, kept.x, None, kept.weight_dtype)
    return dx, dw, _column_sum(summed) if kept.bias else None


class LinearMXFP4Function(torch.autograd.Function):
    @staticmethod
    @custom_fwd(device_type="cuda")
    def forward(ctx: Any, x, weight, bias, out_dtype, seed):
        want_dx, want_dw = getattr(ctx, "needs_input_grad", (False, False))[:2]
        y, kept = _train_fwd(x, weight, bias, out_dtype, want_dx, want_dw)
        ctx.save_for_backward(seed, kept.x and kept.x.data, kept.weight and kept.weight.data)
        # (the operands' tensors are kept by autograd, the rest here)
        ctx.kept = kept._replace(x=kept.x and kept.x._replace(data=None),
                                 weight=kept.weight and kept.weight._replace(data=None))
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @custom_bwd(device_type="cuda")
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, dy):
        seed, x, weight = ctx.saved_tensors
        kept = ctx.kept
        kept = kept._replace(x=kept.x and kept.x._replace(data=x), bias=ctx.needs_input_grad[2],
                             weight=kept.weight and kept.weight._replace(data=weight))
        dx, dw, db = linear_mxfp4_bwd(dy, kept, seed=seed)
        return dx, dw, None if db is None else db.to(ctx.bias_dtype), None, None


def linear_mxfp4(x: torch.Tensor, weight: torch.Tensor | MXFP4Operand, bias: torch.Tensor | None = None, *,
                 stochastic: bool = False, seed: torch.Tensor | None = None) -> torch.Tensor:
    """Differentiable ``linear_mxfp4_fwd`` with the gradients of ``linear_mxfp4_bwd`` (straight through the
    roundings). stochastic: the output's gradient is rounded stochastically, by ``seed`` or one drawn from
    torch's generator (a captured graph draws a new one each replay). Under autocast the output of an fp32 x is
    in the autocast dtype. An operand as the weight carries no gradient, and x must not ask for one. There is no
    forward-mode derivative: dual tensors are refused."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(linear_mxfp4, x, weight, bias, stochastic=stochastic, seed=seed)
    out_dtype = x.dtype
    if x.dtype == torch.float32 and torch.is_autocast_enabled("cuda"):
        out_dtype = torch.get_autocast_dtype("cuda")
    if isinstance(weight, MXFP4Operand):
        if (torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad))) or _has_tangent(x, bias):
            raise ValueError("linear_mxfp4: gradients need the weight itself, not an operand made of it")
        return linear_mxfp4_fwd(x, weight, bias, out_dtype=out_dtype)
    if stochastic and seed is None and torch.is_grad_enabled():
        _on_one_gpu(x)
        seed = DROPOUT_SEEDS.take(x.device)
    if seed is not None:
        _check_seed(seed, x, "linear_mxfp4")
    return apply(LinearMXFP4Function, x, weight, bias, out_dtype, seed if stochastic else None)


class LinearMXFP4(nn.Linear):
    """``nn.Linear`` (same parameters and state-dict keys) as ``linear_mxfp4`` on the GPU, stochastic rounding of
    the output's gradient in training. ``keep_weight`` lays the weight out once for calls that record no
    gradient."""

    _kept: MXFP4Operand | None = None

    @torch.no_grad()
    def keep_weight(self, keep: bool = True) -> None:
        """Calls that record no gradient use the weight as it is now, laid out here, until ``keep_weight(False)``."""
        self._kept = mxfp4_operand(self.weight) if keep else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not x.is_cuda:
            return super().forward(x)
        if self._kept is not None and not torch.is_grad_enabled() and not _has_tangent(self.weight):
            return linear_mxfp4(x, self._kept, self.bias)
        return linear_mxfp4(x, self.weight, self.bias, stochastic=True)


# ---- attention over keys and values in 4 bits ----------------------------------------------
def _in_place(t: torch.Tensor) -> bool:
    return t.stride(3) == 1 and all(s % 16 == 0 for s in _strides(t)) and t.data_ptr() % 16 == 0


def cross_attention_mxfp4_fwd(q: torch.Tensor, kv: MXFP4, *, key_lengths: torch.Tensor | None = None,
                              key_mask: torch.Tensor | None = None,
                              scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``conditioning.cross_attention_fwd`` over keys and values in MXFP4: (out [B, Lq, H, D], lse [B, H, Lq]).

    q [B, Lq, H, D] in bf16 or fp16, kv of the shape [B, Lk, 2, G, D] (keys, then values:
    ``quantize_mxfp4`` of what ``cross_attention_kv`` takes), D a multiple of 32 up to 128, G dividing H.
    Products are those of q's dtype, to which the probabilities are rounded; scores, softmax and sums are fp32. With
    fp16, a value of the cache beyond fp16's range is an infinity (one that was quantised from fp16 is exact). Any strides with dense heads whose
    data lies in multiples of 16 bytes are read in place (``expand`` over the batch, a part of a longer
    cache), others through a copy. Lengths, mask and what hidden keys hold: as there."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(cross_attention_mxfp4_fwd, q, kv, key_lengths=key_lengths, key_mask=key_mask,
                               scale=scale)
    done = _fast().mxfp4_attention(q, kv.data, kv.scales, key_lengths, key_mask, scale)
    if done is not None:
        return done
    _check_mxfp4(kv, "cross attention")
    if q.ndim != 4 or kv.data.ndim != 5 or kv.data.shape[2] != 2:
        raise ValueError("cross attention: q is [batch, tokens, heads, head_dim], kv [batch, tokens, 2, heads, "
                         f"head_dim], got {tuple(q.shape)} and {tuple(kv.shape)}")
    (b, lq, h, d), (bk, lk, _, g, dk) = q.shape, kv.shape
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"cross attention: bf16 or fp16 queries, got {q.dtype}")
    if bk != b or dk != d:
        raise ValueError(f"cross attention: q {tuple(q.shape)} and kv {tuple(kv.shape)} do not go together")
    if d == 0 or d % BLOCK or d > 128:
        raise ValueError(f"cross attention: head_dim {d} is not a multiple of {BLOCK} up to 128")
    if g <= 0 or h <= 0 or h % g:
        raise ValueError(f"cross attention: {h} query heads over {g} key/value heads")
    _on_one_gpu(q, kv.data)
    k = kv.data[:, :, 0]
    lengths, mask = _check_masks(q, k, key_lengths, key_mask)
    number = _scale_of(scale, d)
    q = _rows(q)
    data, scales = kv
    if not (_in_place(data[:, :, 0]) and _in_place(data[:, :, 1])):
        data = data.contiguous() if not data.is_contiguous() else data.clone()
    if scales.stride(4) != 1 and scales.shape[4] > 1:
        scales = scales.contiguous()
    parts = [(t[:, :, i]) for i in (0, 1) for t in (data, scales)]      # keys: data, scales; values
    out = q.new_empty((b, lq, h, d))
    lse = q.new_empty((b, h, lq), dtype=torch.float32)
    if out.numel() == 0:
        return out, lse
    desc = _DESC.pack(q.data_ptr(), *(t.data_ptr() for t in parts), out.data_ptr(), lse.data_ptr(), _ptr(lengths),
                      _ptr(mask), 0 if mask is None else mask.stride(0), *_strides(q),
                      *(s for t in parts for s in _strides(t)), _DT[q.dtype], b, lq, lk, h, g, d, number)
    n = _lib.query("dpa_cross_attention_mxfp4_workspace_bytes", desc)
    ws = _workspace(n, q.device)
    _call("dpa_cross_attention_mxfp4", desc, _ptr(ws), n, q)
    return out, lse


def cross_attention_mxfp4(q: torch.Tensor, kv: MXFP4, *, key_lengths: torch.Tensor | None = None,
                          key_mask: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """``cross_attention_mxfp4_fwd``'s first output, for sampling and serving: it has no gradient, and refuses
    queries that ask for one or carry a tangent. Under autocast fp32 queries are rounded to the autocast dtype first."""
    if (torch.is_grad_enabled() and q.requires_grad) or _has_tangent(q):
        raise ValueError("cross attention over MXFP4 keys and values has no gradient")
    if q.dtype == torch.float32 and torch.is_autocast_enabled("cuda"):
        q = q.to(torch.get_autocast_dtype("cuda"))
    return cross_attention_mxfp4_fwd(q, kv, key_lengths=key_lengths, key_mask=key_mask, scale=scale)[0]
