"""A U-Net conditioned on text: the model of ``unet`` with a token embedding and, behind its
attention levels, blocks of cross attention to the prompt's states, on the operators of
``conditioning``. The reference's U-Net (diffusion/unet.py:245-388) is unconditional; without a
prompt this model computes what ``unet.UNet`` does.

Parameters of the base model keep their names, so a checkpoint of it loads with ``strict=False``,
and the blocks' output projections start at zero, so that the first step is the base model's.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn

from . import conditioning as C
from .layer_norm import layer_norm_bf16
from .layer_norm import supported as ln_supported
from .mxfp4 import BLOCK, MXFP4, LinearMXFP4, cross_attention_mxfp4, quantize_mxfp4
from .unet import UNet, UNetConfig


@dataclass
class TextConfig:
    vocab: int
    width: int
    p_drop: float = 0.1         # of the embeddings and of the blocks' outputs
    padding_idx: int = 0        # takes no part in attention and learns nothing
    mxfp4: bool = False         # the blocks' projections multiply 4-bit operands (``mxfp4.LinearMXFP4``)


class TextEmbedding(nn.Module):
    """tokens [B, L] -> states [B, L, width] in bf16: sqrt(width) weight[token], dropout in
    training. The weight stays in fp32, as its gradient does."""

    def __init__(self, text: TextConfig):
        super().__init__()
        self.text = text
        self.weight = nn.Parameter(torch.randn(text.vocab, text.width) / math.sqrt(text.width))
        with torch.no_grad():
            self.weight[text.padding_idx].zero_()

    def forward(self, tokens: torch.Tensor, dropout: bool = True) -> torch.Tensor:
        return C.embedding(tokens, self.weight, scale=math.sqrt(self.text.width),
                           padding_idx=self.text.padding_idx, p_drop=self.text.p_drop,
                           training=self.training and dropout, out_dtype=torch.bfloat16)


class CrossAttentionBlock(nn.Module):
    """x + dropout(out(cross_attention(q(norm(x)), kv(states)))) over the image's tokens."""

    def __init__(self, channels: int, text: TextConfig, heads: int):
        super().__init__()
        if channels % heads or channels // heads % 8 or channels // heads > 128:
            raise ValueError(f"cross attention block: {channels} channels over {heads} heads")
        self.heads, self.p_drop = heads, text.p_drop
        self.norm = nn.LayerNorm(channels)
        linear = LinearMXFP4 if text.mxfp4 else nn.Linear
        self.q = linear(channels, channels, bias=False)
        self.kv = linear(text.width, 2 * channels, bias=False)
        self.out = linear(channels, channels, bias=False)
        nn.init.zeros_(self.out.weight)

    def project(self, states: torch.Tensor) -> torch.Tensor:
        """Keys and values [B, L, 2, heads, head_dim] of the states; a sampler keeps them over its
        steps."""
        b, l, _ = states.shape
        return self.kv(states).view(b, l, 2, self.heads, self.norm.weight.numel() // self.heads)

    def forward(self, x: torch.Tensor, kv: torch.Tensor | MXFP4, key_mask: torch.Tensor | None) -> torch.Tensor:
        b, c, h, w = x.shape
        seq = x.permute(0, 2, 3, 1).reshape(b, h * w, c)
        y = layer_norm_bf16(seq, self.norm) if ln_supported(c) else self.norm(seq)
        q = self.q(y).view(b, h * w, self.heads, -1)
        o = (cross_attention_mxfp4 if isinstance(kv, MXFP4) else C.cross_attention_kv)(q, kv, key_mask=key_mask)
        o = self.out(o.view(b, h * w, c)).to(seq.dtype)
        y = C.dropout(o, self.p_drop, training=self.training, residual=seq)
        return y.reshape(b, h, w, c).permute(0, 3, 1, 2)


class TextUNet(UNet):
    """``UNet`` with cross attention behind the stages at ``attn_resolutions`` and the middle one.
    Runs under autocast to bf16 on the GPU, as the base model's GPU path does.

    The prompt is an argument of the call or, where the caller knows images and timesteps only
    (``ddpm.DiffusionWrapper``, a captured step), ``prompt``: a tensor of tokens [B, L] that may be
    written between calls."""

    prompt: torch.Tensor | None = None
    _kept: tuple | None = None

    def __init__(self, config: UNetConfig, text: TextConfig):
        super().__init__(config)
        self.text = TextEmbedding(text)
        self.cross = nn.ModuleDict()
        last = len(config.scales) - 1
        for i in range(last):
            if config.in_resolution >> i in config.attn_resolutions:
                here, below = (config.base_hidden * config.scales[j] for j in (i, i + 1))
                self.cross[f"down{i}"] = CrossAttentionBlock(below, text, config.n_heads)
                self.cross[f"up{last - i}"] = CrossAttentionBlock(here, text, config.n_heads)
        self.cross["mid"] = CrossAttentionBlock(config.base_hidden * config.scales[-1], text, config.n_heads)

    def _dropouts(self) -> int:
        n = super()._dropouts()
        if self.training and self.text.text.p_drop > 0.0:
            n += 1 + len(self.cross)
        if self.text.text.mxfp4 and torch.is_grad_enabled():       # stochastic rounding of gradients
            n += sum(isinstance(m, LinearMXFP4) for m in self.cross.modules())
        return n

    def _after_stage(self, name: str, act: torch.Tensor) -> torch.Tensor:
        if self._kv is None or name not in self.cross:
            return act
        return self.cross[name](act, self._kv(name), self._seen)

    _kv = None
    _seen: torch.Tensor | None = None

    @torch.no_grad()
    def keep_prompt(self, tokens: torch.Tensor | None, bits: int = 16) -> None:
        """For sampling: every block's keys and values of these prompts, formed once (without dropout) and
        used by the calls without a prompt of their own until the next ``keep_prompt`` (None: no longer).
        They are of the weights as they are now, and carry no gradient: training steps (calls in training
        mode that record one) take ``prompt``. bits=4: in MXFP4 (heads of a multiple of 32), for calls that
        record no gradient."""
        if bits not in (16, 4):
            raise ValueError(f"keep_prompt: keys and values in 16 or 4 bits, got {bits}")
        if bits == 4 and any(b.norm.weight.numel() // b.heads % BLOCK for b in self.cross.values()):
            raise ValueError(f"keep_prompt: 4 bits need heads of a multiple of {BLOCK}")
        self._kept = None
        if tokens is not None:
            with torch.autocast("cuda", dtype=torch.bfloat16):
                states = self.text(tokens, dropout=False)
                kept = {name: block.project(states) for name, block in self.cross.items()}
                if bits == 4:
                    kept = {name: quantize_mxfp4(kv) for name, kv in kept.items()}
                self._kept = kept, tokens != self.text.text.padding_idx

    def keep_weights(self, keep: bool = True) -> None:
        """For sampling with ``TextConfig.mxfp4``: the blocks' weights as they are now, laid out once for the calls
        that record no gradient, until ``keep_weights(False)``."""
        for m in self.cross.modules():
            if isinstance(m, LinearMXFP4):
                m.keep_weight(keep)

    def _forward(self, x: torch.Tensor, t: torch.Tensor) -> torch.Tensor:
        tokens = self._tokens if self._tokens is not None else self.prompt
        training = self.training and torch.is_grad_enabled()
        if self._tokens is None and self._kept is not None and not training:
            kept, self._seen = self._kept
            self._kv = kept.__getitem__
        elif tokens is not None:
            states = self.text(tokens)
            self._seen = tokens != self.text.text.padding_idx
            self._kv = lambda name: self.cross[name].project(states)
        try:
            return super()._forward(x, t)
        finally:
            self._kv = self._seen = None

    _tokens: torch.Tensor | None = None

    def forward(self, x: torch.Tensor, t: torch.Tensor, tokens: torch.Tensor | None = None) -> torch.Tensor:
        self._tokens = tokens
        try:
            return super().forward(x, t)
        finally:
            self._tokens = None
