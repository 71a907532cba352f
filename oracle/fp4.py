"""The 4-bit paged cache on the CPU in float64: quantisation, layout, and the values it stands for.

Written from the format's definition (include/msattn.h): e2m1 elements, 32 of a row sharing the
power of two 2^e for which the largest magnitude lies in (3.5, 7] 2^e. The reference has no such
cache; tests/test_fp4_oracle.py pins this module by hand-computed answers.
"""
from __future__ import annotations

import numpy as np
import torch

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
TILE, BLOCK = 16, 32


def quantise(x: torch.Tensor) -> tuple[np.ndarray, np.ndarray]:
    """(codes uint8 [.., D], scale bytes uint8 [.., D / 32]) of rows x [.., D]."""
    v = x.double().numpy()
    blocks = v.reshape(*v.shape[:-1], -1, BLOCK)
    bad = ~np.isfinite(blocks).all(axis=-1, keepdims=True)
    v = np.where(bad, 0.0, blocks)
    top = np.abs(v).max(axis=-1, keepdims=True)
    e = np.full(top.shape, -126)
    # the smallest exponent with top <= 7 * 2^e
    for k in range(-126, 126):
        e = np.where((e == k) & (top > 7.0 * 2.0 ** k), min(k + 1, 125), e)
    y = np.abs(v) / 2.0 ** e.astype(float)
    codes = np.zeros(y.shape, dtype=np.uint8)
    for i in range(7):  # past the middle of two levels, or on it where the upper one is even
        mid = (LEVELS[i] + LEVELS[i + 1]) / 2
        codes += ((y > mid) | ((y == mid) & (i % 2 == 1))).astype(np.uint8)
    codes |= np.where(np.signbit(blocks) & ~bad, 8, 0).astype(np.uint8)
    scale = np.where(bad, 255, e + 127).astype(np.uint8)
    return codes.reshape(x.shape), scale[..., 0]


def values(codes: np.ndarray, scale: np.ndarray) -> np.ndarray:
    """Float64 values of codes [.., D] under scale bytes [.., D / 32]."""
    x = np.where(codes & 8, -1.0, 1.0) * LEVELS[codes & 7]
    two = np.where(scale == 255, np.nan, 2.0 ** (scale.astype(float) - 127))
    return (x.reshape(*x.shape[:-1], -1, BLOCK) * two[..., None]).reshape(x.shape)


def pack(codes: np.ndarray, scale: np.ndarray, is_values: bool) -> torch.Tensor:
    """The uint8 cache of codes [blocks, block_size, heads, D] and scales [.., D / 32]."""
    nb, bs, H, D = codes.shape
    out = np.zeros((nb, H, bs // TILE, 17 * D // 2), dtype=np.uint8)
    pair = codes[..., 0::2] | (codes[..., 1::2] << 4)  # [nb, bs, H, D / 2]
    for t in range(bs // TILE):
        for s in range(TILE):
            for i in range(D // 2):
                at = 64 * (i // 4) + 4 * s + i % 4 if is_values else s * (D // 2) + i
                out[:, :, t, at] = pair[:, t * TILE + s, :, i]
            for b in range(D // BLOCK):
                out[:, :, t, 8 * D + b * TILE + s] = scale[:, t * TILE + s, :, b]
    return torch.from_numpy(out)


def unpack(cache: torch.Tensor, is_values: bool) -> tuple[np.ndarray, np.ndarray]:
    """(codes, scale bytes) of a cache: pack's inverse."""
    c = cache.cpu().numpy()
    nb, H, tiles, nbytes = c.shape
    D = nbytes * 2 // 17
    codes = np.zeros((nb, tiles * TILE, H, D), dtype=np.uint8)
    scale = np.zeros((nb, tiles * TILE, H, D // BLOCK), dtype=np.uint8)
    for t in range(tiles):
        for s in range(TILE):
            for i in range(D // 2):
                at = 64 * (i // 4) + 4 * s + i % 4 if is_values else s * (D // 2) + i
                codes[:, t * TILE + s, :, 2 * i] = c[:, :, t, at] & 15
                codes[:, t * TILE + s, :, 2 * i + 1] = c[:, :, t, at] >> 4
            for b in range(D // BLOCK):
                scale[:, t * TILE + s, :, b] = c[:, :, t, 8 * D + b * TILE + s]
    return codes, scale
