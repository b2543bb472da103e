"""MXFP4 layers: the W8A8 layers' shapes and calls on 4-bit weights (format:
``minisgl_amd.kernel.mxfp4``).

``LinearMXFP4`` stands where the reference's linear layers stand
(python/minisgl/layers/linear.py:13-127): ``weight`` uint8 [N, 16 *
ceil(K / 32)] (two e2m1 codes per byte), ``weight_scale`` uint8 [ceil(K / 512),
N, 16] (one power-of-two scale per 32 elements, laid out for the matrix
instructions) and ``bias`` bf16 [N] or None.  Merged projections (q|k|v,
gate|up) concatenate their rows before ``load_mxfp4_weight`` or
``load_float_weight``.  One GPU, as the W8A8 layers.
"""

from __future__ import annotations

from typing import List, Optional, Tuple, Union

import torch

from ..kernel import (
    gated_mlp_mxfp4,
    gated_mlp_quantized_mxfp4,
    gemm_mxfp4,
    linear_mxfp4,
    mxfp4_tile_scales,
    quant_mxfp4,
    rmsnorm_quant_mxfp4,
)
from .base import BaseOP
from .norm import _rows


def _bf16_with_codes_of(w: torch.Tensor) -> torch.Tensor:
    """bf16 values that quantize to the codes and scales of the float tensor w:
    truncated, the last bit set where anything was dropped.  That keeps every
    exponent, so the scales, and the side of every midpoint between two
    levels (its last bf16 bit is 0).  Rounding to nearest would put 1.2500001 on
    the midpoint 1.25 and from there on the wrong level.  Past fp32's range:
    infinity."""
    if w.dtype == torch.bfloat16:
        return w
    if w.dtype in (torch.float16, torch.float32):
        bits = w.float().view(torch.int32)
    else:  # the same step from 64 bits to 32
        w = w.double()
        v = w.float()
        near = v.double()
        bits = v.view(torch.int32) - ((near.abs() > w.abs()) & v.isfinite()).int()
        bits |= ((near != w) & ~v.isinf()).int()
    return ((bits >> 16) | ((bits & 0xFFFF) != 0).int()).to(torch.int16).view(torch.bfloat16)


class LinearMXFP4(BaseOP):
    """``output_size`` a number of rows, or the list of a merged layer's."""

    def __init__(self, input_size: int, output_size: Union[int, List[int]], has_bias: bool = False):
        n = output_size if isinstance(output_size, int) else sum(output_size)
        self.input_size, self.output_size = input_size, n
        self.weight = torch.empty(n, (input_size + 31) // 32 * 16, dtype=torch.uint8)
        self.weight_scale = torch.empty((input_size + 511) // 512, n, 16, dtype=torch.uint8)
        self.bias = torch.empty(n, dtype=torch.bfloat16) if has_bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """bf16 [..., K] -> bf16 [..., N]."""
        return linear_mxfp4(x, self.weight, self.weight_scale, self.bias)

    def forward_quantized(self, codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
        """The product of rows that are quantized already (``RMSNormQuantMXFP4``)."""
        return gemm_mxfp4(codes, scale, self.weight, self.weight_scale, self.bias)

    def load_float_weight(self, w: torch.Tensor, bias: Optional[torch.Tensor] = None) -> None:
        """Quantize a float [N, K] weight (any float type, one rounding) on the
        device into this layer; the bias is rounded to bf16."""
        if w.shape != (self.output_size, self.input_size):
            raise ValueError(f"weight {tuple(w.shape)}, expected {(self.output_size, self.input_size)}")
        self.weight, self.weight_scale = quant_mxfp4(_bf16_with_codes_of(w).contiguous())
        self._load_bias(bias)

    def load_mxfp4_weight(self, codes: torch.Tensor, scale: torch.Tensor, bias: Optional[torch.Tensor] = None) -> None:
        """Take a quantized weight with plain scale rows: codes uint8 [N, 16 *
        ceil(K / 32)], scale bytes uint8 [N, ceil(K / 32)]."""
        blocks = (self.input_size + 31) // 32
        if codes.dtype != torch.uint8 or codes.shape != self.weight.shape:
            raise ValueError(f"codes {tuple(codes.shape)}, expected uint8 {tuple(self.weight.shape)}")
        if scale.dtype != torch.uint8 or scale.shape != (self.output_size, blocks):
            raise ValueError(f"scale {tuple(scale.shape)}, expected uint8 {(self.output_size, blocks)}")
        self.weight, self.weight_scale = codes.contiguous(), mxfp4_tile_scales(scale)
        self._load_bias(bias)

    def _load_bias(self, bias: Optional[torch.Tensor]) -> None:
        if bias is not None:
            if bias.shape != (self.output_size,):
                raise ValueError(f"bias {tuple(bias.shape)}, expected {(self.output_size,)}")
            self.bias = bias.to(torch.bfloat16).contiguous()


class GatedMLPMXFP4(BaseOP):
    """GatedMLP (python/minisgl/models/utils.py:25-50) on MXFP4 weights."""

    def __init__(self, hidden_size: int, intermediate_size: int, hidden_act: str = "silu"):
        if hidden_act not in ("silu", "gelu"):
            raise ValueError(f"Unsupported activation function: {hidden_act}")
        self.gate_up_proj = LinearMXFP4(hidden_size, [intermediate_size, intermediate_size])
        self.down_proj = LinearMXFP4(intermediate_size, hidden_size)
        self._act = hidden_act

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        gu, down = self.gate_up_proj, self.down_proj
        return gated_mlp_mxfp4(x, gu.weight, gu.weight_scale, down.weight, down.weight_scale, self._act)

    def forward_quantized(self, codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
        """The MLP of rows that are quantized already (``RMSNormQuantMXFP4``)."""
        gu, down = self.gate_up_proj, self.down_proj
        return gated_mlp_quantized_mxfp4(codes, scale, gu.weight, gu.weight_scale, down.weight, down.weight_scale, self._act)


class RMSNormQuantMXFP4(BaseOP):
    """RMSNormFused whose output is the MXFP4 input of a linear: ``forward(x,
    residual)`` returns (codes, scale, residual), as ``RMSNormQuant``."""

    def __init__(self, size: int, eps: float) -> None:
        self.eps = eps
        self.weight = torch.empty(size, dtype=torch.bfloat16)

    def forward(
        self, x: torch.Tensor, residual: Optional[torch.Tensor] = None
    ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        x2 = _rows(x)
        if residual is None:
            codes, scale = rmsnorm_quant_mxfp4(x2, self.weight, self.eps)
            return codes, scale, x
        r2 = _rows(residual)
        codes, scale = rmsnorm_quant_mxfp4(x2, self.weight, self.eps, residual=r2)
        if not residual.is_contiguous():
            residual.copy_(r2.view(residual.shape))
        return codes, scale, residual


__all__ = ["GatedMLPMXFP4", "LinearMXFP4", "RMSNormQuantMXFP4"]
