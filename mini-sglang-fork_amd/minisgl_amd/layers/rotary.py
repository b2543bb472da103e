"""Rotary position embedding (python/minisgl/layers/rotary.py): the layer
between the qkv product and attention, with the per-head norms of Qwen3
(python/minisgl/layers/attention.py:49-53) in the same launch if given."""

from __future__ import annotations

import math
from typing import Any, Dict, Optional, Tuple

import torch

from ..kernel import rotary_cos_sin, rotary_qk
from .base import StateLessOP


def rotary_frequencies(
    rotary_dim: int, base: float, scaling: Optional[Dict[str, Any]] = None, max_position: int = 0
) -> Tuple[torch.Tensor, float]:
    """(inverse frequencies fp64 [rotary_dim / 2], factor on cos and sin).

    ``scaling`` is a model's rope_scaling: None, or a dict with ``rope_type``
    (or ``type``) and its numbers:

    * ``default``: f_i = base^(-2 i / d);
    * ``linear``: f_i / factor;
    * ``dynamic``: base grows so that ``max_position`` positions fit (NTK):
      base (factor L / L0 - factor + 1)^(d / (d - 2)), L0 =
      original_max_position_embeddings, L = max(max_position, L0);
    * ``llama3``: waves longer than L0 / low_freq_factor are divided by
      factor, those shorter than L0 / high_freq_factor kept, a linear blend
      in L0 / wavelength between;
    * ``yarn``: frequencies that turn more than beta_fast times over L0 are
      kept, fewer than beta_slow divided by factor, a ramp between (its ends
      on whole indices unless ``truncate`` is false); cos and sin times attention_factor (0.1 ln(factor) + 1, or the ratio of the
      mscale terms where both are given).
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not base > 1:
        raise ValueError(f"base must be above 1, got {base}")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    scaling = scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in ("default", "linear", "dynamic", "llama3", "yarn"):
        raise ValueError(f"unsupported rope scaling {kind!r}")

    def need(name: str) -> float:
        if scaling.get(name) is None:
            raise ValueError(f"rope scaling {kind!r} needs {name}")
        return float(scaling[name])

    if kind == "dynamic":
        factor, original = need("factor"), need("original_max_position_embeddings")
        if rotary_dim <= 2:
            raise ValueError("dynamic rope scaling needs rotary_dim > 2")
        length = max(float(max_position), original)
        base = base * (factor * length / original - (factor - 1)) ** (rotary_dim / (rotary_dim - 2))
    f = float(base) ** (-i / rotary_dim)
    if kind in ("default", "dynamic"):
        return f, 1.0
    factor = need("factor")
    if factor <= 0:
        raise ValueError("rope scaling: factor must be positive")
    if kind == "linear":
        return f / factor, 1.0
    original = need("original_max_position_embeddings")
    if kind == "llama3":
        low, high = need("low_freq_factor"), need("high_freq_factor")
        if not low < high:
            raise ValueError("rope scaling 'llama3': low_freq_factor must be below high_freq_factor")
        blend = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return f * blend + f / factor * (1 - blend), 1.0

    def dim_of(turns: float) -> float:  # the (real) index whose frequency turns so often over the original context
        return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = dim_of(float(scaling.get("beta_fast") or 32)), dim_of(float(scaling.get("beta_slow") or 1))
    if scaling.get("truncate", True):
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, rotary_dim - 1)
    ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
    f = f / factor * ramp + f * (1 - ramp)

    def mscale(weight: float) -> float:
        return 0.1 * weight * math.log(factor) + 1.0 if factor > 1 else 1.0

    if scaling.get("attention_factor") is not None:
        return f, float(scaling["attention_factor"])
    if scaling.get("mscale") and scaling.get("mscale_all_dim"):
        return f, mscale(float(scaling["mscale"])) / mscale(float(scaling["mscale_all_dim"]))
    return f, mscale(1.0)


class RotaryEmbedding(StateLessOP):
    """``forward(positions, query, key)`` rotates query [T, Hq * D or Hq, D]
    and key in place and returns them.  The cos/sin table of ``max_position``
    positions is built once per device, by ``prepare`` or the first
    ``forward`` (which must not be under graph capture)."""

    def __init__(
        self,
        head_size: int,
        rotary_dim: int,
        max_position: int,
        base: float,
        scaling: Optional[Dict[str, Any]] = None,
        interleaved: bool = False,
    ) -> None:
        if not 0 < rotary_dim <= head_size:
            raise ValueError(f"rotary_dim {rotary_dim} must lie in (0, head_size {head_size}]")
        if max_position <= 0:
            raise ValueError("max_position must be positive")
        self.head_size, self.max_position, self.interleaved = head_size, max_position, interleaved
        self._frequencies, self._scale = rotary_frequencies(rotary_dim, base, scaling, max_position)
        self._tables: Dict[int, torch.Tensor] = {}

    def prepare(self, device: torch.device) -> torch.Tensor:
        """The table on ``device``, built if it is not there yet."""
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError("the W8A8 HIP path needs GPU tensors (no CPU fallback)")
        index = torch.cuda.current_device() if dev.index is None else dev.index
        table = self._tables.get(index)
        if table is None:
            with torch.cuda.device(index):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("RotaryEmbedding: call prepare() before the capture")
                table = rotary_cos_sin(self._frequencies.cuda(), self.max_position, self._scale)
                torch.cuda.current_stream().synchronize()  # any stream may read it from here on
            self._tables[index] = table
        return table

    def forward(
        self,
        positions: torch.Tensor,
        query: torch.Tensor,
        key: torch.Tensor,
        q_norm: Optional[Any] = None,
        k_norm: Optional[Any] = None,
    ) -> Tuple[torch.Tensor, torch.Tensor]:
        """``q_norm`` / ``k_norm``: the ``RMSNorm`` layers of the heads (the
        same eps), applied before the rotation."""
        if not query.is_cuda:
            raise ValueError("the W8A8 HIP path needs GPU tensors (no CPU fallback)")
        if q_norm is not None and k_norm is not None and q_norm.eps != k_norm.eps:
            raise ValueError("q_norm and k_norm must have the same eps")
        norm = q_norm if q_norm is not None else k_norm
        rotary_qk(
            self._heads(query),
            self._heads(key),
            positions,
            self.prepare(query.device),
            interleaved=self.interleaved,
            q_weight=None if q_norm is None else q_norm.weight,
            k_weight=None if k_norm is None else k_norm.weight,
            eps=0.0 if norm is None else norm.eps,
        )
        return query, key

    def _heads(self, x: torch.Tensor) -> torch.Tensor:
        """x [T, heads * D] or [T, heads, D] as [T, heads, D]."""
        D = self.head_size
        if x.dim() == 3 and x.shape[2] == D:
            return x
        if x.dim() == 2 and x.shape[1] % D == 0:
            return x.view(x.shape[0], x.shape[1] // D, D)
        raise ValueError(f"query and key: [T, heads * {D}] or [T, heads, {D}], got {tuple(x.shape)}")


__all__ = ["RotaryEmbedding", "rotary_frequencies"]
