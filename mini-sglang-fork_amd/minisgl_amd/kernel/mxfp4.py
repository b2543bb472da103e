"""MXFP4 operators: 4-bit e2m1 elements with one power-of-two scale per 32.

A quantized matrix [rows, K] is two uint8 tensors:

* ``codes`` [rows, 16 * ceil(K / 32)]: two elements per byte, the even one in
  the low half, a last partial block filled with zeros;
* ``scale`` [ceil(K / 512), rows, 16]: byte ``e + 127`` of each block's scale
  2^e (255: NaN), in the order in which the matrix instructions read them:
  of the 16 blocks of 512 elements, block ``8 t + 2 g + s`` is byte
  ``4 g + 2 t + s``; bytes of blocks past K are 0.  ``mxfp4_tile_scales``
  brings the plain [rows, ceil(K / 32)] form into it (a weight's scales,
  once, when it is loaded), ``mxfp4_row_scales`` back.

Quantization (section 6.3 of the OCP microscaling specification): ``e =
floor(log2(amax)) - 2`` clamped to [-127, 127], elements rounded to nearest
even and saturated at 6 * 2^e; a zero block gets byte 0, a block with NaN or
an infinity byte 255.  Products accumulate in fp32.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .lib import check, load
from .ops import _ACT, _call_workspace, _device_of, _need, _on_gpu, _ptr, _same_device, _stream


def _codes_width(K: int) -> int:
    return (K + 31) // 32 * 16


def _tiles(K: int) -> int:
    return (K + 511) // 512


def _empty(rows: int, K: int, like: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    codes = torch.empty(rows, _codes_width(K), dtype=torch.uint8, device=like.device)
    scale = torch.empty(_tiles(K), rows, 16, dtype=torch.uint8, device=like.device)
    return codes, scale


def mxfp4_tile_scales(rows: torch.Tensor) -> torch.Tensor:
    """Scale bytes [rows, blocks] -> the layout [ceil(blocks / 16), rows, 16]
    of the products (a copy; any device)."""
    _need(rows.dtype == torch.uint8 and rows.dim() == 2 and rows.shape[1] > 0, "scales: uint8 [rows, blocks]")
    n, blocks = rows.shape
    tiles = (blocks + 15) // 16
    full = torch.zeros((n, tiles * 16), dtype=torch.uint8, device=rows.device)
    full[:, :blocks].copy_(rows)
    return full.view(n, tiles, 2, 4, 2).permute(1, 0, 3, 2, 4).reshape(tiles, n, 16)


def mxfp4_row_scales(scale: torch.Tensor, K: int) -> torch.Tensor:
    """The inverse of ``mxfp4_tile_scales``: scale bytes [rows, ceil(K / 32)]."""
    _need(scale.dtype == torch.uint8 and scale.dim() == 3 and scale.shape[2] == 16 and scale.shape[0] == _tiles(K),
          "scales: uint8 [ceil(K / 512), rows, 16]")
    tiles, n, _ = scale.shape
    rows = scale.view(tiles, n, 4, 2, 2).permute(1, 0, 3, 2, 4).reshape(n, tiles * 16)
    return rows[:, : (K + 31) // 32].contiguous()


def quant_mxfp4(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """bf16 [M, K] (any row stride, any K) -> (codes, scale)."""
    _on_gpu(x)
    _need(x.dtype == torch.bfloat16 and x.dim() == 2 and x.shape[1] > 0, "quant_mxfp4: x must be bf16 [M, K]")
    _need(x.stride(1) == 1 or x.shape[1] == 1, "quant_mxfp4: last dim must be contiguous")
    M, K = x.shape
    _need(M <= 1 or x.stride(0) >= K, "quant_mxfp4: rows must not overlap")
    codes, scale = _empty(M, K, x)
    if M > 0:
        with _device_of(x):
            check(load().mw8_quant_mxfp4_bf16(_ptr(x), M, K, max(x.stride(0), K), _ptr(codes), _ptr(scale), _stream(x)))
    return codes, scale


def act_and_mul_quant_mxfp4(x: torch.Tensor, activation: str = "silu") -> Tuple[torch.Tensor, torch.Tensor]:
    """bf16 [R, 2d] (gate | up) -> (codes, scale) of bf16(act(gate) * up) [R, d]."""
    _on_gpu(x)
    _need(activation in _ACT, f"unsupported activation {activation}")
    _need(x.dtype == torch.bfloat16 and x.dim() == 2 and x.is_contiguous(), "x: bf16 [R, 2d] contiguous")
    R, two_d = x.shape
    _need(two_d > 0 and two_d % 2 == 0, "x: bf16 [R, 2d]")
    codes, scale = _empty(R, two_d // 2, x)
    if R > 0:
        with _device_of(x):
            check(load().mw8_act_and_mul_quant_mxfp4_bf16(_ptr(x), R, two_d, _ACT[activation], _ptr(codes), _ptr(scale),
                                                          _stream(x)))
    return codes, scale


def rmsnorm_quant_mxfp4(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float,
    residual: Optional[torch.Tensor] = None,
    y: Optional[torch.Tensor] = None,
    return_y: bool = False,
):
    """``rmsnorm_quant`` with the MXFP4 quantizer: bf16 x [M, H] -> (codes,
    scale[, bf16 y [M, H]]) of the normalized rows, bit-identical to
    ``quant_mxfp4`` of its y.  ``residual`` is added first and updated in
    place; ``y`` may be ``x``; x, residual and y share no memory otherwise.
    H % 8 == 0, H <= 32768."""
    _one_gpu(x, weight, residual, y)
    _need(x.dtype == torch.bfloat16 and x.dim() == 2 and x.is_contiguous(), "x: bf16 [M, H] contiguous")
    M, H = x.shape
    _need(H > 0, "x: bf16 [M, H]")
    _need(weight.dtype == torch.bfloat16 and weight.shape == (H,) and weight.is_contiguous(), "weight: bf16 [H]")
    if residual is not None:
        _need(residual.dtype == torch.bfloat16 and residual.shape == (M, H) and residual.is_contiguous(),
              "residual: bf16 [M, H] contiguous")
        _need(M == 0 or residual.data_ptr() != x.data_ptr(), "residual must not be x")
    if return_y and y is None:
        y = torch.empty((M, H), dtype=torch.bfloat16, device=x.device)
    if y is not None:
        _need(y.dtype == torch.bfloat16 and y.shape == (M, H) and y.is_contiguous(), "y: bf16 [M, H]")
        _need(M == 0 or residual is None or y.data_ptr() != residual.data_ptr(), "y must not be residual")
    codes, scale = _empty(M, H, x)
    if M > 0:
        with _device_of(x):
            check(load().mw8_rmsnorm_quant_mxfp4_bf16(_ptr(x), _ptr(residual), _ptr(weight), float(eps), M, H, _ptr(codes),
                                                      _ptr(scale), _ptr(y), _stream(x)))
    return (codes, scale, y) if y is not None else (codes, scale)


def _one_gpu(*ts: Optional[torch.Tensor]) -> None:
    """Every tensor on one GPU (``_on_gpu`` and ``_same_device`` in one pass
    over device indices: an eager decode call is bound by its host time)."""
    index = ts[0].get_device()
    for t in ts:
        if t is not None and (t.get_device() != index or index < 0):
            _on_gpu(*ts)
            _same_device(*ts)


def _check_operand(name: str, codes: torch.Tensor, scale: torch.Tensor, K: Optional[int]) -> int:
    """Checks a quantized matrix and returns its rows; K None: a whole number
    of blocks, as wide as the codes."""
    if not (codes.dtype == torch.uint8 and codes.dim() == 2 and codes.is_contiguous() and codes.shape[1] > 0
            and codes.shape[1] % 16 == 0):
        raise ValueError(f"{name}: codes uint8 [rows, 16 * ceil(K / 32)] contiguous")
    rows, width = codes.shape
    k = width * 2 if K is None else K
    if not (k > 0 and width == _codes_width(k)):
        raise ValueError(f"{name}: codes of {width} bytes a row do not hold K = {K}")
    if not (scale.dtype == torch.uint8 and scale.shape == (_tiles(k), rows, 16) and scale.is_contiguous()):
        raise ValueError(f"{name}: scale uint8 [{_tiles(k)}, {rows}, 16] contiguous (mxfp4_tile_scales)")
    return rows


def dequant_mxfp4(codes: torch.Tensor, scale: torch.Tensor, K: Optional[int] = None) -> torch.Tensor:
    """The values of a quantized matrix, bf16 [rows, K] (K None: every block whole)."""
    _one_gpu(codes, scale)
    M = _check_operand("dequant_mxfp4", codes, scale, K)
    K = codes.shape[1] * 2 if K is None else K
    y = torch.empty((M, K), dtype=torch.bfloat16, device=codes.device)
    if M > 0:
        with _device_of(codes):
            check(load().mw8_dequant_mxfp4_bf16(_ptr(codes), _ptr(scale), M, K, _ptr(y), _stream(codes)))
    return y


def _check_bias_out(bias, out, M: int, N: int) -> None:
    if bias is not None:
        _need(bias.dtype == torch.bfloat16 and bias.shape == (N,) and bias.is_contiguous(), "bias: bf16 [N]")
    if out is not None:
        _need(out.dtype == torch.bfloat16 and out.shape == (M, N) and out.is_contiguous(), "out: bf16 [M, N]")
        if bias is not None:  # (blocks read it while others write)
            b, o = bias.data_ptr(), out.data_ptr()
            _need(b + 2 * N <= o or o + 2 * M * N <= b, "out must not overlap bias")


def gemm_mxfp4(
    q: torch.Tensor,
    s_a: torch.Tensor,
    w: torch.Tensor,
    s_w: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """y bf16 [M, N] = bf16(A W^T + bias[n]) of quantized A [M, K], W [N, K]."""
    _one_gpu(q, s_a, w, s_w, bias, out)
    M, N = _check_operand("A", q, s_a, None), _check_operand("W", w, s_w, None)
    _need(q.shape[1] == w.shape[1], "A/W K mismatch")
    _need(N > 0, "W: at least one row")
    _check_bias_out(bias, out, M, N)
    y = out if out is not None else torch.empty((M, N), dtype=torch.bfloat16, device=q.device)
    if M > 0:
        with _device_of(q):
            _gemm(q, s_a, w, s_w, bias, y, M, N)
    return y


def _gemm(q, s_a, w, s_w, bias, y, M: int, N: int) -> None:
    """The product's launch, its tensors checked and their device current."""
    lib, K = load(), q.shape[1] * 2
    need = 0 if M <= 16 else lib.mw8_gemm_mxfp4_workspace_bytes(M, N, K)
    ws = _call_workspace(need, q)
    check(lib.mw8_gemm_mxfp4_bf16(q.data_ptr(), s_a.data_ptr(), w.data_ptr(), s_w.data_ptr(), _ptr(bias), y.data_ptr(),
                                  M, N, K, _ptr(ws), need, _stream(q)))


def gemm_act_mxfp4(
    q: torch.Tensor, s_a: torch.Tensor, w: torch.Tensor, s_w: torch.Tensor, activation: str = "silu"
) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes, scale) of act(gate) * up [M, I] for the quantized A [M, K] and
    gate_up weight [2I, K]: ``gemm_mxfp4`` and ``act_and_mul_quant_mxfp4`` in one
    launch, with their bits but for the order of the product's fp32 additions
    (``gemm_mxfp4`` picks among kernels and K splits).  I % 32 == 0."""
    _one_gpu(q, s_a, w, s_w)
    _need(activation in _ACT, f"unsupported activation {activation}")
    M, N = _check_operand("A", q, s_a, None), _check_operand("W", w, s_w, None)
    _need(q.shape[1] == w.shape[1], "A/W K mismatch")
    _need(N > 0 and N % 64 == 0, "W: 2I rows, I a multiple of 32")
    codes, scale = _empty(M, N // 2, q)
    if M > 0:
        with _device_of(q):
            check(load().mw8_gemm_act_mxfp4(_ptr(q), _ptr(s_a), _ptr(w), _ptr(s_w), _ACT[activation], _ptr(codes),
                                            _ptr(scale), M, N // 2, q.shape[1] * 2, _stream(q)))
    return codes, scale


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [M, K] with contiguous, separate rows (x itself, or a copy)."""
    return x if x.stride(1) == 1 and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()


def linear_mxfp4(
    x: torch.Tensor, w: torch.Tensor, s_w: torch.Tensor, bias: Optional[torch.Tensor] = None
) -> torch.Tensor:
    """bf16 x [..., K] times a quantized weight [N, K]: y bf16 [..., N].  The
    rows of x are quantized (``quant_mxfp4``) on the way: a few rows (8 at
    most, 2 at K = 5120) inside the product's launch, with the same bits."""
    _one_gpu(x, w, s_w, bias)
    _need(x.dtype == torch.bfloat16 and x.dim() >= 1 and x.shape[-1] > 0, "linear_mxfp4: x must be bf16 [..., K]")
    N = _check_operand("W", w, s_w, x.shape[-1])
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    x2 = _rows(x2)
    M, K = x2.shape
    _check_bias_out(bias, None, M, N)
    ldx = K if M <= 1 else x2.stride(0)
    # (the one launch reads x through a 32-bit view: rows less than 2^26 elements apart)
    if 0 < M <= 8 and x2.data_ptr() % 16 == 0 and (M == 1 or (ldx % 8 == 0 and ldx < 1 << 26)):
        lib = load()
        with _device_of(x):
            if lib.mw8_linear_bf16_mxfp4_supported(M, N, K):
                y = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
                check(lib.mw8_linear_bf16_mxfp4(x2.data_ptr(), ldx, w.data_ptr(), s_w.data_ptr(), _ptr(bias),
                                                y.data_ptr(), M, N, K, _stream(x)))
                return y if x.dim() == 2 else y.view(*x.shape[:-1], N)
    y = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    if M > 0:
        codes, scale = quant_mxfp4(x2)
        with _device_of(x):
            _gemm(codes, scale, w, s_w, bias, y, M, N)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)


def gated_mlp_mxfp4(
    x: torch.Tensor,
    w_gate_up: torch.Tensor,
    s_gate_up: torch.Tensor,
    w_down: torch.Tensor,
    s_down: torch.Tensor,
    activation: str = "silu",
) -> torch.Tensor:
    """down(act(gate(x)) * up(x)) on quantized weights gate_up [2I, H] (gate
    rows first) and down [H', I]: bf16 x [..., H] -> bf16 [..., H'].  gate,
    up and their product are rounded to bf16 before the product is
    quantized for down.  Large batches run gate_up, activation and
    quantizer as one launch (``gemm_act_mxfp4``)."""
    _one_gpu(x, w_gate_up, s_gate_up, w_down, s_down)
    _need(x.dtype == torch.bfloat16 and x.dim() >= 1 and x.shape[-1] > 0, "gated_mlp_mxfp4: x must be bf16 [..., H]")
    inter, N = _check_mlp(x.shape[-1], w_gate_up, s_gate_up, w_down, s_down, activation)
    x2 = _rows(x if x.dim() == 2 else x.reshape(-1, x.shape[-1]))
    M, H = x2.shape
    y = _mlp(x2, H if M <= 1 else x2.stride(0), None, None, w_gate_up, s_gate_up, w_down, s_down, activation, M, H, inter, N)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)


def gated_mlp_quantized_mxfp4(
    codes: torch.Tensor,
    scale: torch.Tensor,
    w_gate_up: torch.Tensor,
    s_gate_up: torch.Tensor,
    w_down: torch.Tensor,
    s_down: torch.Tensor,
    activation: str = "silu",
) -> torch.Tensor:
    """``gated_mlp_mxfp4`` of rows that are quantized already (codes, scale
    of [M, H], as ``rmsnorm_quant_mxfp4`` gives them): bf16 [M, H']."""
    _one_gpu(codes, scale, w_gate_up, s_gate_up, w_down, s_down)
    M, K = _check_operand("x", codes, scale, None), codes.shape[1] * 2
    inter, N = _check_mlp(K, w_gate_up, s_gate_up, w_down, s_down, activation)
    return _mlp(None, 0, codes, scale, w_gate_up, s_gate_up, w_down, s_down, activation, M, K, inter, N)


def _check_mlp(K: int, w_gate_up, s_gate_up, w_down, s_down, activation: str) -> Tuple[int, int]:
    """(I, output size) of a gated MLP on rows of K."""
    _need(activation in _ACT, f"unsupported activation {activation}")
    rows = _check_operand("gate_up", w_gate_up, s_gate_up, K)
    _need(rows > 0 and rows % 2 == 0, "gate_up: 2I rows")
    N = _check_operand("down", w_down, s_down, rows // 2)
    _need(N > 0, "down: at least one row")
    return rows // 2, N


def _mlp(x, ldx: int, codes, scale, w_gate_up, s_gate_up, w_down, s_down, activation: str, M: int, H: int, inter: int,
         N: int) -> torch.Tensor:
    """The MLP's launches in one call (an eager call of each is bound by host
    time in decode batches: 4 launches 35 us one by one)."""
    like, lib = w_down, load()
    y = torch.empty(M, N, dtype=torch.bfloat16, device=like.device)
    if M > 0:
        with _device_of(like):
            need = lib.mw8_gated_mlp_mxfp4_workspace_bytes(x is None, M, H, inter, N)
            ws = _call_workspace(need, like)
            check(lib.mw8_gated_mlp_mxfp4(_ptr(x), ldx, _ptr(codes), _ptr(scale), w_gate_up.data_ptr(), s_gate_up.data_ptr(),
                                          w_down.data_ptr(), s_down.data_ptr(), _ACT[activation], y.data_ptr(), M, H, inter, N,
                                          _ptr(ws), need, _stream(like)))
    return y


__all__ = [
    "act_and_mul_quant_mxfp4",
    "dequant_mxfp4",
    "gated_mlp_mxfp4",
    "gated_mlp_quantized_mxfp4",
    "gemm_act_mxfp4",
    "gemm_mxfp4",
    "linear_mxfp4",
    "mxfp4_row_scales",
    "mxfp4_tile_scales",
    "quant_mxfp4",
    "rmsnorm_quant_mxfp4",
]
