"""Operators that condition the U-Net on text, on the HIP library's kernels: token embedding
(``dpa_embedding_*``), cross attention of image tokens to an encoder's states
(``dpa_cross_attention_*``) and dropout (``dpa_dropout``).

Each comes as functions of one launch sequence per direction (``*_fwd``, ``*_bwd``, which record
nothing, for captured steps and samplers) and as a differentiable function (``cross_attention``,
``cross_attention_kv``, ``embedding``, ``dropout``). The reference's U-Net (diffusion/unet.py) is
unconditional and has no counterpart. GPU tensors only; there is no fallback.

Dropout masks come from the counter hash of the GroupNorm kernels: 16 bits per element of
splitmix64(seed + (index / 4) * golden ratio) against floor(p * 2^16), the seed an int64 tensor of
one element on the device (``gn_silu.new_dropout_seed``). No mask is stored; the backward
recomputes it.
"""
from __future__ import annotations

import math
import struct
from typing import Any, NamedTuple

import torch
from torch.amp.autocast_mode import custom_bwd, custom_fwd

from . import _lib
from .eager import apply
from .gn_silu import DROPOUT_SEEDS

_DT = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}     # DPA_DTYPE_*
_MAX_HEAD_DIM = 128
_MAX_WIDTH = 1 << 20        # of a row of the embedding

# DpaCrossAttention of include/dpa_fp8.h: 11 pointers, the mask's stride, 6 x 3 strides, 7 sizes,
# the scale
_DESC = struct.Struct("=11Qq18q7if")
_DESC_HEAD, _DESC_TAIL = struct.Struct("=11Q"), struct.Struct("=q18q7if")


class _General:
    """Stands for the native calls where they are not built: every call goes the general way."""

    def __getattr__(self, name):
        return lambda *args: None


_FAST: Any = None


def _fast():
    """``csrc/fast_calls.cpp``: each of its functions does a whole call on operands that need no
    conversion, and returns None for any other, which the code behind it copies or refuses."""
    global _FAST
    if _FAST is None:
        _FAST = _lib.fast_calls() or _General()
    return _FAST


@torch.compiler.disable
def _between_graphs(function, *args, **kwargs):
    """``function`` under torch.compile: the graph ends before the call, and nothing in it is traced (Dynamo
    does not know the native calls)."""
    return function(*args, **kwargs)


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _on_one_gpu(*tensors: torch.Tensor | None) -> None:
    first = tensors[0].get_device()
    for t in tensors:
        if t is not None and (first < 0 or t.get_device() != first):
            raise ValueError(f"expected GPU tensors on one device, got {t.device} and {tensors[0].device}")


# ---- cross attention ---------------------------------------------------------------------
def _strides(t: torch.Tensor) -> tuple[int, int, int]:
    """Element strides of batch, token and head; those of dimensions of one element are 0."""
    return tuple(0 if n <= 1 else s for n, s in zip(t.shape[:3], t.stride()[:3]))


def _in_place(t: torch.Tensor) -> bool:
    """Whether the kernels read t where it is (its 16-B alignment apart): dense head_dim, strides of
    whole 16 B."""
    return t.stride(3) == 1 and all(s % 8 == 0 for s in _strides(t))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as the kernels read it, else a dense copy."""
    if _in_place(t) and t.data_ptr() % 16 == 0:
        return t
    return t.contiguous() if not t.is_contiguous() else t.clone()


def _check_qkv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError("cross attention: q, k, v are [batch, tokens, heads, head_dim], got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"cross attention: q {tuple(q.shape)}, k {tuple(k.shape)} and "
                         f"v {tuple(v.shape)} do not go together")
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"cross attention: bf16 or fp16 operands of one dtype, got {q.dtype}, "
                         f"{k.dtype}, {v.dtype}")
    d, h, g = q.shape[3], q.shape[2], k.shape[2]
    if d <= 0 or d % 8 or d > _MAX_HEAD_DIM:
        raise ValueError(f"cross attention: head_dim {d} is not a multiple of 8 up to {_MAX_HEAD_DIM}")
    if g <= 0 or h <= 0 or h % g:
        raise ValueError(f"cross attention: {h} query heads over {g} key/value heads")
    _on_one_gpu(q, k, v)


def _check_masks(q, k, key_lengths, key_mask):
    b, lk = q.shape[0], k.shape[1]
    if key_lengths is not None:
        if key_lengths.shape != (b,) or key_lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"cross attention: key_lengths are int32 or int64 [{b}], got "
                             f"{key_lengths.dtype} {tuple(key_lengths.shape)}")
        _on_one_gpu(q, key_lengths)
        if key_lengths.dtype != torch.int32:
            # (clamped first: a length past 2^31 keeps its meaning)
            key_lengths = key_lengths.clamp(0, lk).to(torch.int32)
        key_lengths = key_lengths.contiguous()
    if key_mask is not None:
        if key_mask.shape != (b, lk) or key_mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"cross attention: key_mask is bool or uint8 [{b}, {lk}], got "
                             f"{key_mask.dtype} {tuple(key_mask.shape)}")
        _on_one_gpu(q, key_mask)
        if key_mask.stride(1) != 1 and lk > 1:
            key_mask = key_mask.contiguous()
    return key_lengths, key_mask


def _scale_of(scale: float | None, head_dim: int) -> float:
    if scale is None:
        return 1.0 / math.sqrt(head_dim)
    scale = float(scale)
    if not 0.0 < scale < 2.3e38:        # (scale log2(e) is finite in fp32)
        raise ValueError(f"cross attention: scale {scale} is not positive and below 2.3e38")
    return scale


_NONE3 = (0, 0, 0)


class _Call(NamedTuple):
    """The operands of a call as the kernels read them, checked, and what follows from their layout."""
    q: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    lengths: torch.Tensor | None
    mask: torch.Tensor | None
    dout: torch.Tensor | None
    tail: bytes         # DpaCrossAttention behind its pointers

    def describe(self, out, lse, dq=None, dk=None, dv=None) -> bytes:
        return _DESC_HEAD.pack(self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), out.data_ptr(),
                               lse.data_ptr(), _ptr(self.lengths), _ptr(self.mask), _ptr(self.dout),
                               _ptr(dq), _ptr(dk), _ptr(dv)) + self.tail


def _attention_call(q, k, v, lengths, mask, scale, dout=None, dk=None, dv=None) -> _Call:
    _check_qkv(q, k, v)
    if dout is not None:
        if dout.shape != q.shape or dout.dtype != q.dtype:
            raise ValueError(f"cross attention: dout {dout.dtype} {tuple(dout.shape)} is not q's "
                             f"{q.dtype} {tuple(q.shape)}")
        _on_one_gpu(q, dout)
        dout = _rows(dout)
    lengths, mask = _check_masks(q, k, lengths, mask)
    (b, lq, h, d), (lk, g) = q.shape, k.shape[1:3]
    number = _scale_of(scale, d)
    q, k, v = _rows(q), _rows(k), _rows(v)
    strides = [_NONE3 if t is None else _strides(t) for t in (q, k, v, dout, dk, dv)]
    tail = _DESC_TAIL.pack(0 if mask is None else mask.stride(0), *(s for t in strides for s in t),
                           _DT[q.dtype], b, lq, lk, h, g, d, number)
    return _Call(q, k, v, lengths, mask, dout, tail)


def _workspace(nbytes: int, device) -> torch.Tensor | None:
    return torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None


def cross_attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                        key_lengths: torch.Tensor | None = None,
                        key_mask: torch.Tensor | None = None,
                        scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """softmax(scale q k^T) v over the keys that take part, and log sum exp of the scores.

    q [B, Lq, H, D], k and v [B, Lk, G, D] in bf16 or fp16, D a multiple of 8 up to 128, G dividing
    H (query head h reads key head h // (H / G)). Any strides with dense heads are read in place
    when they are multiples of 8 elements -- halves of a packed projection, ``expand`` over the
    batch -- others through a dense copy. A key takes part below key_lengths[b] (int32 or int64
    [B], clamped to [0, Lk]) and where key_mask ([B, Lk], bool or uint8) is true; what keys hold
    that do not changes nothing (rows from the length on are not read, rows that the mask hides may be). A
    query without any gets 0, and -inf as its log sum exp. scale: 1 / sqrt(D) by default, positive.
    Returns (out [B, Lq, H, D], lse [B, H, Lq] fp32)."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(cross_attention_fwd, q, k, v, key_lengths=key_lengths, key_mask=key_mask, scale=scale)
    done = _fast().attention_fwd(q, k, v, key_lengths, key_mask, scale)
    if done is not None:
        return done
    call = _attention_call(q, k, v, key_lengths, key_mask, scale)
    b, lq, h, d = q.shape
    out = q.new_empty((b, lq, h, d))
    lse = q.new_empty((b, h, lq), dtype=torch.float32)
    if out.numel() == 0:
        return out, lse
    desc = call.describe(out, lse)
    n = _lib.query("dpa_cross_attention_fwd_workspace_bytes", desc)
    ws = _workspace(n, q.device)
    _lib.call("dpa_cross_attention_fwd", desc, _ptr(ws), n, _lib.current_stream(q))
    return out, lse


def _attention_bwd(dout, q, k, v, out, lse, key_lengths, key_mask, scale, dk, dv):
    """(dq, dk, dv); dk and dv: None (not formed), True (a new dense tensor) or where to write them."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(_attention_bwd, dout, q, k, v, out, lse, key_lengths, key_mask, scale, dk, dv)
    done = _fast().attention_bwd(dout, q, k, v, out, lse, key_lengths, key_mask, scale, dk, dv)
    if done is not None:
        return done
    if dk is True:
        dk, dv = k.new_empty(k.shape), k.new_empty(k.shape)
    call = _attention_call(q, k, v, key_lengths, key_mask, scale, dout, dk, dv)
    b, lq, h, d = q.shape
    if out.shape != q.shape or out.dtype != q.dtype or out.get_device() != q.get_device():
        raise ValueError(f"cross attention: out {out.dtype} {tuple(out.shape)} on {out.device} is not "
                         f"q's {q.dtype} {tuple(q.shape)} on {q.device}")
    if lse.shape != (b, h, lq) or lse.dtype != torch.float32 or lse.get_device() != q.get_device():
        raise ValueError(f"cross attention: lse is fp32 [{b}, {h}, {lq}] on {q.device}, got "
                         f"{lse.dtype} {tuple(lse.shape)} on {lse.device}")
    out, lse = out.contiguous(), lse.contiguous()
    if out.data_ptr() % 16:
        out = out.clone()
    dq = q.new_empty((b, lq, h, d))
    if b == 0 or (dq.numel() == 0 and (dk is None or dk.numel() == 0)):
        return dq, dk, dv
    desc = call.describe(out, lse, dq, dk, dv)
    n = _lib.query("dpa_cross_attention_bwd_workspace_bytes", desc)
    ws = _workspace(n, q.device)
    _lib.call("dpa_cross_attention_bwd", desc, _ptr(ws), n, _lib.current_stream(q))
    return dq, dk, dv


def cross_attention_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                        out: torch.Tensor, lse: torch.Tensor, *,
                        key_lengths: torch.Tensor | None = None,
                        key_mask: torch.Tensor | None = None, scale: float | None = None
                        ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv) of ``cross_attention_fwd`` from its outputs and the gradient of out; dk and dv
    [B, Lk, G, D] summed over the query heads of a key head, zero for keys that take no part.
    Deterministic."""
    return _attention_bwd(dout, q, k, v, out, lse, key_lengths, key_mask, scale, True, True)


class CrossAttention(torch.autograd.Function):
    @staticmethod
    @custom_fwd(device_type="cuda")
    def forward(ctx: Any, q, k, v, key_lengths, key_mask, scale):
        out, lse = cross_attention_fwd(q, k, v, key_lengths=key_lengths, key_mask=key_mask,
                                       scale=scale)
        ctx.save_for_backward(q, k, v, out, lse, key_lengths, key_mask)
        ctx.scale = scale
        return out

    @staticmethod
    @custom_bwd(device_type="cuda")
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, dout):
        q, k, v, out, lse, lengths, mask = ctx.saved_tensors
        keys = True if ctx.needs_input_grad[1] or ctx.needs_input_grad[2] else None
        return (*_attention_bwd(dout, q, k, v, out, lse, lengths, mask, ctx.scale, keys, keys),
                None, None, None)


class CrossAttentionKV(torch.autograd.Function):
    """CrossAttention over packed keys and values, whose gradient is written packed too."""

    @staticmethod
    @custom_fwd(device_type="cuda")
    def forward(ctx: Any, q, kv, key_lengths, key_mask, scale):
        out, lse = cross_attention_fwd(q, kv[:, :, 0], kv[:, :, 1], key_lengths=key_lengths,
                                       key_mask=key_mask, scale=scale)
        ctx.save_for_backward(q, kv, out, lse, key_lengths, key_mask)
        ctx.scale = scale
        return out

    @staticmethod
    @custom_bwd(device_type="cuda")
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, dout):
        q, kv, out, lse, lengths, mask = ctx.saved_tensors
        dkv = torch.empty(kv.shape, device=kv.device, dtype=kv.dtype) if ctx.needs_input_grad[1] else None
        dk, dv = (None, None) if dkv is None else (dkv[:, :, 0], dkv[:, :, 1])
        dq, _, _ = _attention_bwd(dout, q, kv[:, :, 0], kv[:, :, 1], out, lse, lengths, mask, ctx.scale, dk, dv)
        return dq, dkv, None, None, None


def _autocast(*tensors: torch.Tensor) -> tuple[torch.Tensor, ...]:
    """Operands as a matrix product under autocast takes them."""
    if torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        return tuple(t.to(dt) if t.dtype == torch.float32 else t for t in tensors)
    return tensors


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                    key_lengths: torch.Tensor | None = None,
                    key_mask: torch.Tensor | None = None,
                    scale: float | None = None) -> torch.Tensor:
    """Differentiable ``cross_attention_fwd`` (its first output). Under autocast fp32 operands are
    rounded to the autocast dtype first."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(cross_attention, q, k, v, key_lengths=key_lengths, key_mask=key_mask, scale=scale)
    q, k, v = _autocast(q, k, v)
    return apply(CrossAttention, q, k, v, key_lengths, key_mask, scale)


def cross_attention_kv(q: torch.Tensor, kv: torch.Tensor, *,
                       key_lengths: torch.Tensor | None = None,
                       key_mask: torch.Tensor | None = None,
                       scale: float | None = None) -> torch.Tensor:
    """``cross_attention`` over keys and values side by side, kv [B, Lk, 2, G, D] (a projection of
    the encoder's states to 2 G D columns). A sampler projects them once and keeps kv over its
    steps."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(cross_attention_kv, q, kv, key_lengths=key_lengths, key_mask=key_mask, scale=scale)
    if kv.ndim != 5 or kv.shape[2] != 2:
        raise ValueError(f"cross attention: kv is [batch, tokens, 2, heads, head_dim], got {tuple(kv.shape)}")
    q, kv = _autocast(q, kv)
    return apply(CrossAttentionKV, q, kv, key_lengths, key_mask, scale)


# ---- dropout -----------------------------------------------------------------------------
def _check_p(p: float, what: str) -> float:
    p = float(p)
    if not 0.0 <= p < 1.0 or not struct.unpack("f", struct.pack("f", p))[0] < 1.0:
        raise ValueError(f"{what}: p {p} is not in [0, 1)")
    return p


def _check_seed(seed, like: torch.Tensor, what: str) -> None:
    if seed is None or seed.dtype != torch.int64 or seed.numel() != 1:
        raise ValueError(f"{what}: the seed is an int64 tensor of one element on the device")
    _on_one_gpu(like, seed)


def _dense(t: torch.Tensor) -> torch.Tensor:
    if t.is_contiguous() or (t.ndim == 4 and t.is_contiguous(memory_format=torch.channels_last)):
        return t
    return t.contiguous()


def _in_order_of(t: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """t with x's memory order (x dense)."""
    if x.is_contiguous():
        return t.contiguous()
    return t.contiguous(memory_format=torch.channels_last)


def dropout_fwd(x: torch.Tensor, p: float, seed: torch.Tensor, *,
                residual: torch.Tensor | None = None) -> torch.Tensor:
    """residual + keep x / (1 - p) (residual: a tensor of x's shape and dtype, or none), formed in
    fp32 and rounded once. x is bf16, fp16 or fp32. An element's place in memory is its index for
    the mask (dense or channels-last tensors as they are, others as their dense copy); the result
    has x's layout. A dropped element counts as 0 whatever it holds."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(dropout_fwd, x, p, seed, residual=residual)
    y = _fast().dropout(x, p, seed, residual)
    if y is not None:
        return y
    if x.dtype not in _DT:
        raise ValueError(f"dropout: bf16, fp16 or fp32, got {x.dtype}")
    p = _check_p(p, "dropout")
    _on_one_gpu(x)
    _check_seed(seed, x, "dropout")
    x = _dense(x)
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"dropout: residual {residual.dtype} {tuple(residual.shape)} is not x's "
                             f"{x.dtype} {tuple(x.shape)}")
        _on_one_gpu(x, residual)
        residual = _in_order_of(residual, x)
    y = torch.empty_like(x)
    _lib.call("dpa_dropout", x.data_ptr(), _ptr(residual), y.data_ptr(), _DT[x.dtype], x.numel(),
              seed.data_ptr(), p, _lib.current_stream(x))
    return y


def dropout_bwd(dy: torch.Tensor, p: float, seed: torch.Tensor) -> torch.Tensor:
    """The gradient of x from dy in x's memory order (the residual's is dy itself)."""
    return dropout_fwd(dy, p, seed)


class Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x, p, seed, residual):
        y = dropout_fwd(x, p, seed, residual=residual)
        ctx.save_for_backward(seed)
        ctx.p = p
        ctx.order = torch.contiguous_format if y.is_contiguous() else torch.channels_last
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, dy):
        (seed,) = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0]:
            dx = dropout_bwd(dy.contiguous(memory_format=ctx.order), ctx.p, seed)
        return dx, None, None, dy if ctx.needs_input_grad[3] else None


def dropout(x: torch.Tensor, p: float = 0.5, *, training: bool = True,
            residual: torch.Tensor | None = None, seed: torch.Tensor | None = None) -> torch.Tensor:
    """Differentiable ``dropout_fwd``. seed: drawn from torch's generator when not given (a captured
    graph draws a new one each replay). Without training, or with p = 0, x (+ residual)."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(dropout, x, p, training=training, residual=residual, seed=seed)
    p = _check_p(p, "dropout")
    if not training or p == 0.0:
        return x if residual is None else residual + x
    if seed is None:
        _on_one_gpu(x)
        seed = DROPOUT_SEEDS.take(x.device)
    return apply(Dropout, x, p, seed, residual)


# ---- embedding ---------------------------------------------------------------------------
def _check_embedding(tokens, table_dtype, other_dtype, p_drop, seed, like):
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"embedding: tokens are int32 or int64, got {tokens.dtype}")
    if table_dtype not in _DT or other_dtype not in _DT:
        raise ValueError(f"embedding: bf16, fp16 or fp32, got {table_dtype} and {other_dtype}")
    p_drop = _check_p(p_drop, "embedding")
    _on_one_gpu(like, tokens)
    if p_drop > 0.0:
        _check_seed(seed, like, "embedding")
    return p_drop


def embedding_fwd(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0,
                  p_drop: float = 0.0, seed: torch.Tensor | None = None,
                  out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """scale weight[tokens] in out_dtype (weight's by default), with p_drop > 0 followed by dropout
    (index: the element's place in the output; seed as in ``dropout_fwd``). tokens int32 or int64
    of any shape, weight [V, C] bf16, fp16 or fp32. A token outside [0, V) gives a row of NaN."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(embedding_fwd, tokens, weight, scale=scale, p_drop=p_drop, seed=seed,
                               out_dtype=out_dtype)
    out = _fast().embedding_fwd(tokens, weight, scale, p_drop, seed, out_dtype)
    if out is not None:
        return out
    if weight.ndim != 2 or weight.numel() == 0 or weight.shape[1] > _MAX_WIDTH:
        raise ValueError(f"embedding: the weight is [V, C], C up to {_MAX_WIDTH}, got {tuple(weight.shape)}")
    out_dtype = weight.dtype if out_dtype is None else out_dtype
    p_drop = _check_embedding(tokens, weight.dtype, out_dtype, p_drop, seed, weight)
    v, c = weight.shape
    weight, tokens = weight.contiguous(), tokens.contiguous()
    out = weight.new_empty((*tokens.shape, c), dtype=out_dtype)
    _lib.call("dpa_embedding_fwd", tokens.data_ptr(), tokens.element_size(), weight.data_ptr(),
              _DT[weight.dtype], out.data_ptr(), _DT[out_dtype], tokens.numel(), v, c, float(scale),
              seed.data_ptr() if p_drop > 0.0 else None, p_drop, _lib.current_stream(weight))
    return out


def embedding_bwd(dout: torch.Tensor, tokens: torch.Tensor, num_embeddings: int, *,
                  scale: float = 1.0, padding_idx: int | None = None, p_drop: float = 0.0,
                  seed: torch.Tensor | None = None, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The gradient [num_embeddings, C] of ``embedding_fwd``'s weight in dtype (dout's by default):
    per row the fp32 sum over its tokens, rounded once; zeros for padding_idx. Tokens outside the table
    add nothing. A row's tokens are summed by position, many in pieces of up to 32 whose sums are then
    added: always in the same order."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(embedding_bwd, dout, tokens, num_embeddings, scale=scale, padding_idx=padding_idx,
                               p_drop=p_drop, seed=seed, dtype=dtype)
    dw = _fast().embedding_bwd(dout, tokens, num_embeddings, scale, padding_idx, p_drop, seed, dtype)
    if dw is not None:
        return dw
    if dout.ndim < 1 or dout.shape[:-1] != tokens.shape or dout.shape[-1] == 0 or num_embeddings <= 0:
        raise ValueError(f"embedding: dout {tuple(dout.shape)} does not go with tokens "
                         f"{tuple(tokens.shape)} and {num_embeddings} rows")
    if dout.shape[-1] > _MAX_WIDTH:
        raise ValueError(f"embedding: rows of up to {_MAX_WIDTH}, got {dout.shape[-1]}")
    dtype = dout.dtype if dtype is None else dtype
    p_drop = _check_embedding(tokens, dout.dtype, dtype, p_drop, seed, dout)
    if padding_idx is None:
        padding_idx = -1
    elif not 0 <= padding_idx < num_embeddings:
        raise ValueError(f"embedding: padding_idx {padding_idx} is outside the {num_embeddings} rows")
    c, n = dout.shape[-1], tokens.numel()
    dout, tokens = dout.contiguous(), tokens.contiguous()
    dw = dout.new_empty((num_embeddings, c), dtype=dtype)
    nbytes = _lib.query("dpa_embedding_bwd_workspace_bytes", n, c)
    ws = _workspace(nbytes, dout.device)
    _lib.call("dpa_embedding_bwd", dout.data_ptr(), _DT[dout.dtype], tokens.data_ptr(),
              tokens.element_size(), dw.data_ptr(), _DT[dtype], n, num_embeddings, c, float(scale),
              padding_idx, seed.data_ptr() if p_drop > 0.0 else None, p_drop, _ptr(ws), nbytes,
              _lib.current_stream(dout))
    return dw


class Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, weight, tokens, scale, padding_idx, p_drop, seed, out_dtype):
        out = embedding_fwd(tokens, weight, scale=scale, p_drop=p_drop, seed=seed, out_dtype=out_dtype)
        ctx.save_for_backward(tokens, seed)
        ctx.args = (weight.shape[0], weight.dtype, scale, padding_idx, p_drop)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, dout):
        tokens, seed = ctx.saved_tensors
        v, dtype, scale, padding_idx, p_drop = ctx.args
        dw = embedding_bwd(dout, tokens, v, scale=scale, padding_idx=padding_idx, p_drop=p_drop,
                           seed=seed, dtype=dtype)
        return dw, None, None, None, None, None, None


def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0,
              padding_idx: int | None = None, p_drop: float = 0.0, training: bool = True,
              seed: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Differentiable ``embedding_fwd``; the weight's gradient comes in its own dtype. Dropout only
    with training; seed as in ``dropout``."""
    if torch.compiler.is_dynamo_compiling():
        return _between_graphs(embedding, tokens, weight, scale=scale, padding_idx=padding_idx, p_drop=p_drop,
                               training=training, seed=seed, out_dtype=out_dtype)
    p_drop = _check_p(p_drop, "embedding") if training else 0.0
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f"embedding: padding_idx {padding_idx} is outside the {weight.shape[0]} rows")
    if p_drop > 0.0 and seed is None:
        _on_one_gpu(weight)
        seed = DROPOUT_SEEDS.take(weight.device)
    return apply(Embedding, weight, tokens, float(scale), padding_idx, p_drop,
                 seed if p_drop > 0.0 else None, out_dtype)
