"""The 4-bit form of cache rows in 64 bits (numpy, on the host), from its definition."""

from __future__ import annotations

import numpy as np

NAN_WORD = 0x7E00


def values(codes, words):
    """uint8 codes [..., d / 2] and 16-bit words [..., d / 32] as the values they stand for."""
    codes = np.asarray(codes, np.uint8)
    words = np.asarray(words).astype(np.int64) & 0xFFFF
    c = np.stack([codes & 15, codes >> 4], axis=-1).reshape(*codes.shape[:-1], -1).astype(np.float64)
    scale = (words & 0xFFF0).astype(np.uint16).view(np.float16).astype(np.float64)
    with np.errstate(all="ignore"):
        v = (c - np.repeat(words & 15, 32, axis=-1)) * np.repeat(scale, 32, axis=-1)
        return np.where(np.abs(v) > 65504.0, np.inf * np.sign(v), v)


def quantize(x):
    """(codes uint8 [..., d / 2], words int16 [..., d / 32]) of float64 x [..., d]."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(g).all(axis=-1)
    g = np.clip(np.where(bad[..., None], 0.0, g), -32768.0, 32768.0)
    lo, hi = np.minimum(g.min(axis=-1), 0.0), np.maximum(g.max(axis=-1), 0.0)
    step = (hi - lo) / 15.0
    mantissa, e = np.frexp(step)  # in [0.5, 1): 7 bits are multiples of 2^-7
    up = np.ldexp(np.ceil(mantissa * 128.0), e - 7)
    scale = np.where(step >= 2.0 ** -14, up, np.maximum(np.ceil(step * 2.0 ** 20), 1.0) * 2.0 ** -20)
    zero = np.rint(-lo / scale)
    codes = np.clip(np.rint(g / scale[..., None]) + zero[..., None], 0, 15)
    codes = np.where(bad[..., None], 0, codes).astype(np.uint8).reshape(x.shape)
    words = scale.astype(np.float16).view(np.uint16) | zero.astype(np.uint16)
    words = np.where(bad, NAN_WORD, words).astype(np.uint16).view(np.int16)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), words


def random_cache(rng, *shape, loud=1.0):
    """Codes and words [..., d] of any kind that a cache may hold, values near `loud`, and the values."""
    codes = rng.integers(0, 256, (*shape[:-1], shape[-1] // 2)).astype(np.uint8)
    scale = np.ldexp(rng.integers(64, 128, (*shape[:-1], shape[-1] // 32)) / 64.0, rng.integers(-4, -1, 1)[0]) * loud
    words = scale.astype(np.float16).view(np.uint16) & 0xFFF0 | rng.integers(0, 16, scale.shape).astype(np.uint16)
    words = words.astype(np.uint16).view(np.int16)
    return codes, words, values(codes, words)
