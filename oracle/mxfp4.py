"""CPU restatement (numpy, fp64) of the MXFP4 operators, from their
definitions: block quantizer, scale layout, values, product, gated
activation and RMSNorm before the quantizer.  Test infrastructure only."""

from __future__ import annotations

import math

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def blocks(k: int) -> int:
    return -(-k // 32)


def round_bf16(x: np.ndarray) -> np.ndarray:
    """fp64 -> bf16-valued fp64, round to nearest even (subnormals included)."""
    x = np.asarray(x, np.float64)
    m, e = np.frexp(x)  # |m| in [0.5, 1)
    ulp = np.exp2(np.maximum(e - 8, -133).astype(np.float64))
    with np.errstate(invalid="ignore"):
        y = np.rint(x / ulp) * ulp
    y = np.where(np.abs(y) >= 2.0**128, np.copysign(np.inf, x), y)
    return np.where(np.isfinite(x), y, x)


def nearest_level(a: float) -> int:
    """Code (0..7) of the level nearest to a >= 0; a tie goes to the even code."""
    best = min(range(8), key=lambda i: (abs(LEVELS[i] - a), i & 1))
    return best


def quantize(x: np.ndarray):
    """x [M, K] -> codes (0..15) [M, 32 blocks], scale bytes [M, blocks]."""
    x = np.asarray(x, np.float64)
    M, K = x.shape
    B = blocks(K)
    v = np.zeros((M, B * 32))
    v[:, :K] = x
    v = v.reshape(M, B, 32)
    bad = ~np.isfinite(v).all(2)
    amax = np.where(bad, 1.0, np.abs(np.where(np.isfinite(v), v, 0)).max(2))
    e = np.where(amax > 0, np.frexp(amax)[1] - 1 - 2, -127)
    e = np.clip(e, -127, 127)
    a = np.where(bad[:, :, None], 0.0, v) / np.exp2(e.astype(np.float64))[:, :, None]
    mag = np.abs(a)
    code = np.zeros(a.shape, np.uint8)
    # the midpoint between two levels belongs to the even code
    for i in range(7):
        mid = (LEVELS[i] + LEVELS[i + 1]) / 2
        code += (mag > mid) | ((mag == mid) & (i % 2 == 1))
    code += 8 * np.signbit(a).astype(np.uint8)
    code[bad] = 0
    byte = np.where(bad, 255, e + 127).astype(np.uint8)
    return code.reshape(M, B * 32), byte


def pack(code: np.ndarray) -> np.ndarray:
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


def unpack(packed: np.ndarray) -> np.ndarray:
    out = np.empty((packed.shape[0], packed.shape[1] * 2), np.uint8)
    out[:, 0::2] = packed & 15
    out[:, 1::2] = packed >> 4
    return out


def tile_scales(byte: np.ndarray) -> np.ndarray:
    """[rows, blocks] -> [ceil(blocks / 16), rows, 16], one byte at a time."""
    rows, B = byte.shape
    out = np.zeros((-(-B // 16), rows, 16), np.uint8)
    for b in range(B):
        t, g, s = (b % 16) // 8, (b % 8) // 2, b % 2
        out[b // 16, :, 4 * g + 2 * t + s] = byte[:, b]
    return out


def values(code: np.ndarray, byte: np.ndarray) -> np.ndarray:
    """fp64 values; NaN in the blocks of byte 255."""
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))
    return v * np.repeat(s, 32, axis=1)


def product(a: np.ndarray, w: np.ndarray, bias=None):
    """(A W^T + bias in fp64, the sum of the absolute values of its terms)."""
    y, size = a @ w.T, np.abs(a) @ np.abs(w).T
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    return y, size


def activation(g: np.ndarray, act: str) -> np.ndarray:
    with np.errstate(over="ignore"):
        if act == "silu":
            return g / (1 + np.exp(-g))
    return 0.5 * g * np.vectorize(math.erfc)(-g / math.sqrt(2))


def rmsnorm(x: np.ndarray, w: np.ndarray, eps: float) -> np.ndarray:
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
