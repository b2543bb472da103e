"""Rotary position embedding of q and k on the GPU (the reference calls
flashinfer's apply_rope_with_cos_sin_cache_inplace,
python/minisgl/layers/rotary.py:35-52)."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .lib import check, load
from .mxfp4 import _one_gpu
from .ops import _device_of, _need, _on_gpu, _ptr, _stream

_DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _strides(name: str, t: torch.Tensor) -> Tuple[int, int]:
    """(token, head) strides of t [T, heads, D] with contiguous heads."""
    T, heads, D = t.shape
    ld, hd, one = t.stride()
    if one != 1 and D != 1:
        raise ValueError(f"{name}: last dim must be contiguous")
    if heads <= 1:
        hd = D
    if T <= 1:
        ld = hd * max(heads, 1)
    # heads within a token's span, or tokens within a head's
    if not (hd >= D and ld >= hd * (heads - 1) + D or ld >= D and hd >= ld * (T - 1) + D):
        raise ValueError(f"{name}: rows must not overlap")
    return ld, hd


def rotary_qk(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: torch.Tensor,
    cos_sin: torch.Tensor,
    interleaved: bool = False,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    q_out: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rotates q [T, Hq, D] and k [T, Hk, D] (bf16, fp16 or fp32; views of the
    qkv product as they lie) by the angles of ``positions`` [T] (int32 or
    int64), in place or into ``q_out`` / ``k_out``; returns both outputs.

    ``cos_sin`` fp32 [P, R]: R / 2 cosines, then R / 2 sines per position
    (``rotary_cos_sin``); the first R elements of a head are turned, the rest
    pass.  Pairs are (i, R / 2 + i), or (2 i, 2 i + 1) if ``interleaved``.
    ``q_weight`` / ``k_weight`` [D]: the per-head RMSNorm x / rms(x) * weight
    before the rotation.  All of it in fp32, rounded once.

    A token whose position is negative is padding: its output rows stay as
    they are.  One past the table turns to NaN.  Outputs may be the inputs
    themselves; otherwise no output may overlap an input or the other (views
    of one buffer that share no element are fine); the library refuses it."""
    _one_gpu(q, k, positions, cos_sin, q_weight, k_weight, q_out, k_out)
    _need(q.dtype in _DTYPE and k.dtype == q.dtype, "q and k: bf16, fp16 or fp32, the same")
    _need(q.dim() == 3 and k.dim() == 3 and q.shape[0] == k.shape[0] and q.shape[2] == k.shape[2],
          "q: [T, Hq, D] and k: [T, Hk, D]")
    T, hq, D = q.shape
    hk = k.shape[1]
    _need(positions.shape == (T,) and positions.dtype in (torch.int32, torch.int64) and positions.is_contiguous(),
          "positions: int32 or int64 [T]")
    _need(cos_sin.dtype == torch.float32 and cos_sin.dim() == 2 and cos_sin.is_contiguous() and cos_sin.shape[0] > 0,
          "cos_sin: fp32 [P, R]")
    P, R = cos_sin.shape
    _need(0 < R <= D and R % 2 == 0, "cos_sin: R must be even, positive and at most the head size")
    for w in (q_weight, k_weight):
        _need(w is None or (w.dtype == q.dtype and w.shape == (D,) and w.is_contiguous()), "norm weights: [D], as q")
    q_out = q if q_out is None else q_out
    k_out = k if k_out is None else k_out
    _need(q_out.dtype == q.dtype and q_out.shape == q.shape and k_out.dtype == q.dtype and k_out.shape == k.shape,
          "q_out and k_out: as q and k")
    _need(D <= 8192 and hq + hk < 1 << 26, "q and k: heads of at most 8192 elements, fewer than 2^26 heads")
    if T == 0 or hq + hk == 0:
        return q_out, k_out
    if hq and hk:
        _need(q_out.data_ptr() != k_out.data_ptr(), "q_out and k_out must not overlap")
        _need(q_out.data_ptr() != k.data_ptr() and k_out.data_ptr() != q.data_ptr(), "q_out and k, k_out and q must not overlap")
    qs, ks = _strides("q", q), _strides("k", k)
    qos = qs if q_out is q else _strides("q_out", q_out)
    kos = ks if k_out is k else _strides("k_out", k_out)
    with _device_of(q):
        check(load().mw8_rotary_qk(
            _ptr(q), *qs, hq, _ptr(k), *ks, hk, _ptr(q_out), *qos, _ptr(k_out), *kos, _DTYPE[q.dtype], D, R, int(interleaved), _ptr(positions),
            int(positions.dtype == torch.int64), _ptr(cos_sin), P, _ptr(q_weight), _ptr(k_weight), float(eps), T,
            _stream(q)))
    return q_out, k_out


def rotary_cos_sin(inv_freq: torch.Tensor, positions: int, scale: float = 1.0) -> torch.Tensor:
    """The table of ``rotary_qk``: fp32 [positions, 2 * pairs], cos and sin of
    p * inv_freq[i] (inv_freq fp64 [pairs], the angle in fp64) times ``scale``."""
    _on_gpu(inv_freq)
    _need(inv_freq.dtype == torch.float64 and inv_freq.dim() == 1 and inv_freq.is_contiguous() and 0 < inv_freq.numel() <= 4096,
          "inv_freq: fp64 [pairs], at most 4096")
    _need(positions >= 0, "positions must be >= 0")
    half = inv_freq.numel()
    table = torch.empty((positions, 2 * half), dtype=torch.float32, device=inv_freq.device)
    if positions > 0:
        with _device_of(inv_freq):
            check(load().mw8_rotary_cos_sin(_ptr(inv_freq), half, positions, float(scale), _ptr(table),
                                            _stream(inv_freq)))
    return table


__all__ = ["rotary_cos_sin", "rotary_qk"]
