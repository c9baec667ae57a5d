"""Microscaled 4-bit floating point in plain numpy, 64 bits: the oracle of the tests of quantisation and of the products that read it."""

from __future__ import annotations

import numpy as np

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MIDDLES = (VALUES[:-1] + VALUES[1:]) / 2


def quantize(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes [rows, blocks, 32] 0..15, scale bytes [rows, blocks]) of a float64 matrix whose numbers are float32 or bfloat16 values."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = np.zeros((rows, blocks * 32))
    v[:, :cols] = x
    v = v.reshape(rows, blocks, 32)
    finite = np.isfinite(v).all(axis=2)
    top = np.where(finite[:, :, None], np.abs(v), 0.0).max(axis=2)
    _, exponent = np.frexp(top)                                     # top = m 2^exponent, 0.5 <= m < 1
    s = np.where(top > 0, np.maximum(exponent - 1 - 2 + 127, 0), 0)
    s = np.where(finite, s, 255)
    with np.errstate(invalid="ignore"):
        scaled = np.abs(v) * np.exp2(127.0 - np.minimum(s, 254))[:, :, None]
    # the number of midpoints below it; on a midpoint, of the two values as near the one whose code is even
    scaled = np.where(finite[:, :, None], scaled, 0.0)
    code = np.searchsorted(MIDDLES, scaled, side="left")
    code = np.where(scaled == MIDDLES[np.minimum(code, 6)], code + code % 2, code)
    code = code + 8 * np.signbit(v)
    return np.where(finite[:, :, None], code, 0).astype(np.uint8), s.astype(np.uint8)


def values(codes: np.ndarray, scales: np.ndarray, cols: int) -> np.ndarray:
    factor = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    v = np.where(codes < 8, 1.0, -1.0) * VALUES[codes & 7] * factor[:, :, None]
    return v.reshape(codes.shape[0], -1)[:, :cols]


def unpack(packed: np.ndarray, blocks: int) -> np.ndarray:
    """The codes [rows, blocks, 32] of a matrix of bytes."""
    return np.stack([packed & 15, packed >> 4], axis=2).reshape(packed.shape[0], blocks, 32)


def rounded(x: np.ndarray) -> np.ndarray:
    codes, scales = quantize(x)
    return values(codes, scales, x.shape[1])


def gated(kind: str, g: np.ndarray, u: np.ndarray, limit: float, alpha: float) -> np.ndarray:
    with np.errstate(over="ignore"):
        if kind == "relu":
            return np.maximum(g, 0.0) * u
        if kind == "clamped_swish":
            g, u = np.minimum(g, limit), np.clip(u, -limit, limit)
            return g / (1 + np.exp(-alpha * g)) * (u + 1)
        if kind == "gelu_tanh":
            return 0.5 * g * (1 + np.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3))) * u
        return g / (1 + np.exp(-g)) * u
