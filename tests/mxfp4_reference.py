"""MXFP4 by its definition, in 64 bits on the CPU."""
from __future__ import annotations

import numpy as np
import torch

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = 32


def random_bits(rows: int, cols: int, seed: int) -> np.ndarray:
    """16 bits for each element of a matrix whose rows count whole blocks: splitmix64, four to a hash."""
    pitch = -(-cols // BLOCK) * BLOCK
    with np.errstate(over="ignore"):
        z = np.uint64(seed) + np.arange(rows * pitch // 4, dtype=np.uint64) * np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        z ^= z >> np.uint64(31)
    return z.view("<u2").reshape(rows, pitch)[:, :cols].astype(np.int64)


def quantize(x: torch.Tensor, bits: np.ndarray | None = None) -> tuple[np.ndarray, np.ndarray]:
    """(codes [..., C], scale bytes [..., ceil(C / 32)]) with blocks along the last dimension; codes of a
    block without a value are -1."""
    v = x.detach().cpu().double().numpy()
    c = v.shape[-1]
    pad = -c % BLOCK
    widths = [(0, 0)] * (v.ndim - 1) + [(0, pad)]
    v = np.pad(v, widths).reshape(*v.shape[:-1], (c + pad) // BLOCK, BLOCK)
    amax = np.abs(v).max(-1, keepdims=True)
    none = ~np.isfinite(amax)
    amax = np.where(none, 1.0, amax)
    v = np.where(none, 0.0, v)
    k = np.where(amax > 0, np.frexp(amax)[1] - 1, -200) - 2
    if bits is not None:
        k = np.where(amax > 6.0 * np.exp2(k.astype(float)), k + 1, k)
    k = np.maximum(k, -127)
    size = np.abs(v) / np.exp2(k.astype(float))
    low = np.clip(np.searchsorted(GRID, size, side="right") - 1, 0, 7)
    above = np.append(GRID, 8.0)[low + 1]
    if bits is None:
        near = (size - GRID[low]) - (above - size)
        up = (near > 0) | ((near == 0) & (low % 2 == 1))
    else:
        b = np.pad(bits, widths).reshape(size.shape)
        up = np.floor((size - GRID[low]) / (above - GRID[low]) * 65536) + b >= 65536
    code = np.minimum(low + up, 7) + 8 * (np.signbit(v) & (size >= 0))
    code = np.where(none, -1, code)
    byte = np.where(none, 255, k + 127)[..., 0]
    return code.reshape(*code.shape[:-2], c + pad)[..., :c], byte


def values_of(code: np.ndarray, byte: np.ndarray) -> torch.Tensor:
    """The numbers that codes [..., C] and scale bytes stand for (NaN where there is none)."""
    signed = np.where(code >= 8, -1.0, 1.0) * GRID[np.where(code < 0, 0, code) % 8]
    scale = np.where(byte == 255, np.nan, np.exp2(byte.astype(float) - 127)).repeat(BLOCK, -1)[..., :code.shape[-1]]
    return torch.from_numpy(signed * scale)


def rounded(x: torch.Tensor, along: int = -1, seed: int | None = None) -> torch.Tensor:
    """The values that MXFP4 keeps of the matrix x with blocks along a dimension."""
    bits = None if seed is None else random_bits(*x.shape, seed)
    if along == 0:
        return values_of(*quantize(x.t(), None if bits is None else bits.T)).t().contiguous()
    return values_of(*quantize(x, bits))


def unpack(data: torch.Tensor) -> np.ndarray:
    d = data.cpu().numpy()
    return np.stack((d & 15, d >> 4), -1).reshape(*d.shape[:-1], 2 * d.shape[-1])


def pack(code: np.ndarray) -> torch.Tensor:
    c = code.astype(np.uint8)
    return torch.from_numpy(c[..., ::2] | c[..., 1::2] << 4)
