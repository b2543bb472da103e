"""CPU restatement (numpy, fp64) of the rotary operators.  Test
infrastructure only."""

from __future__ import annotations

import numpy as np


def table(inv_freq: np.ndarray, positions: int, scale: float) -> np.ndarray:
    ang = np.arange(positions, dtype=np.float64)[:, None] * inv_freq[None, :]
    return np.concatenate([np.cos(ang), np.sin(ang)], 1) * scale


def rotate(x, cos_sin, pos, interleaved=False, weight=None, eps=1e-6):
    """x [T, H, D] fp64; pos [T] (every one inside the table)."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    R = cos_sin.shape[1]
    y = x.copy()
    for i in range(R // 2):
        ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, R // 2 + i)
        c, s = cos_sin[pos, i][:, None], cos_sin[pos, R // 2 + i][:, None]
        y[..., ia] = x[..., ia] * c - x[..., ib] * s
        y[..., ib] = x[..., ib] * c + x[..., ia] * s
    return y
