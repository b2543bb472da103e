"""GPU parity of the MXFP4 quantizers against the CPU oracle: codes and scale
bytes equal, over every bf16 value and over shapes, strides and alignments;
the fused forms equal the quantizer of what they quantize."""

import numpy as np
import pytest
import torch

from helpers import announce, f32
from minisgl_amd.kernel import (
    act_and_mul_quant_mxfp4,
    dequant_mxfp4,
    mxfp4_row_scales,
    quant_mxfp4,
    rmsnorm_quant,
    rmsnorm_quant_mxfp4,
)
from oracle import mxfp4 as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _acts(M, K, seed, spread=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=gen)
    x[torch.rand(M, K, generator=gen) < 1e-3] *= 20
    if spread:  # rows and columns over the exponent range
        x = x * torch.exp2(torch.randint(-spread, spread, (M, K), generator=gen).float())
    return x.to(torch.bfloat16)


def _same(got, x):
    """got = (codes, scale) is the oracle's quantization of x (bf16, CPU)."""
    codes, scale = (t.cpu().numpy() for t in got)
    code, byte = orc.quantize(f32(x).astype(np.float64))
    np.testing.assert_array_equal(scale, orc.tile_scales(byte))
    np.testing.assert_array_equal(codes, orc.pack(code))


@pytest.mark.parametrize("M,K", [(1, 1), (1, 31), (1, 32), (2, 33), (1, 5120), (3, 500), (5, 512), (64, 520), (65, 513),
                                 (67, 1000), (130, 1032), (333, 160), (70, 4099), (2, 17408)])
def test_quant_equals_oracle(M, K):
    announce(f"quant_mxfp4 M={M} K={K}")
    x = _acts(M, K, seed=M * 131 + K, spread=6)
    _same(quant_mxfp4(x.to(DEV)), x)


def test_quant_every_bf16_value():
    """Every finite bf16 bit pattern, each beside block maxima that give its
    own scale, one higher and the smallest."""
    announce("quant_mxfp4 every value")
    bits = torch.arange(65536, dtype=torch.int32)
    v = bits.to(torch.int16).view(torch.bfloat16)
    v = v[torch.isfinite(v)]
    n = v.numel()
    rows = []
    for k in (0, 1, 3):  # the block's largest entry: the value times 2^k
        x = torch.zeros(n, 32, dtype=torch.bfloat16)
        x[:, 5] = v
        big = (v.double() * 2.0**k).abs().clamp(max=3.0e38).bfloat16()
        x[:, 20] = big
        rows.append(x)
    x = torch.cat(rows)
    _same(quant_mxfp4(x.to(DEV)), x)


def test_quant_nan_and_infinity():
    announce("quant_mxfp4 NaN / inf / zero blocks")
    x = _acts(70, 1000, seed=5)
    x[3, 7], x[4, 999], x[66, 512], x[66, 40] = float("nan"), float("inf"), float("-inf"), float("nan")
    x[9] = 0
    x[10, :64] = -0.0
    got = quant_mxfp4(x.to(DEV))
    _same(got, x)
    y = dequant_mxfp4(*got, K=1000)
    assert torch.isnan(y[3, :32]).all() and torch.isfinite(y[3, 32:]).all()
    assert torch.isnan(y[4, 992:]).all() and not y[9].any()


@pytest.mark.parametrize("ld,off", [(1024, 0), (1032, 0), (1024, 8), (1024, 3), (1001, 0), (1003, 1)])
@pytest.mark.parametrize("M", [4, 70])
def test_quant_strides_and_alignment(M, ld, off):
    announce(f"quant_mxfp4 strided M={M} ld={ld} off={off}")
    base = _acts(1, M * ld + 16, seed=ld + off)[0]
    x = base.to(DEV)[off:].as_strided((M, 1000), (ld, 1))
    _same(quant_mxfp4(x), x.cpu())


def test_dequant_every_code_and_scale():
    announce("dequant_mxfp4 every code and scale")
    code = np.tile(np.arange(16, dtype=np.uint8), 2)
    codes = np.broadcast_to(orc.pack(code[None]), (256, 16)).copy()
    byte = np.arange(256, dtype=np.uint8)[:, None]
    scale = torch.from_numpy(orc.tile_scales(byte)).to(DEV)
    y = f32(dequant_mxfp4(torch.from_numpy(codes).to(DEV), scale)).astype(np.float64)
    want = orc.round_bf16(orc.values(np.broadcast_to(code, (256, 32)), byte))
    np.testing.assert_array_equal(y, want)
    np.testing.assert_array_equal(np.signbit(y[1:255]), np.signbit(want[1:255]))


@pytest.mark.parametrize("M,K", [(1, 7), (3, 500), (65, 1000), (9, 5120)])
def test_dequant_round_trip(M, K):
    x = _acts(M, K, seed=K, spread=4)
    y = dequant_mxfp4(*quant_mxfp4(x.to(DEV)), K=K)
    code, byte = orc.quantize(f32(x).astype(np.float64))
    np.testing.assert_array_equal(f32(y).astype(np.float64), orc.values(code, byte)[:, :K])
    again = quant_mxfp4(y)  # values of the format quantize to themselves where the maximum keeps its exponent
    z = dequant_mxfp4(*again, K=K)
    assert torch.equal(z, y)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,d", [(1, 32), (3, 33), (1, 17408), (66, 768), (70, 500), (4, 6400)])
def test_act_and_mul_quant(M, d, act):
    """Codes of bf16(act(g) u): the activation's fp32 error (exp, reciprocal,
    erf: under 2^-20 relative to the result, times the product) may move its
    bf16 rounding by one step and a code by its spacing; everything else is
    exact.  So the values are compared with the oracle's on the unrounded
    activation: half a spacing of the code, plus the bf16 rounding."""
    announce(f"act_and_mul_quant_mxfp4 M={M} d={d} {act}")
    x = _acts(M, 2 * d, seed=M + d)
    codes, scale = act_and_mul_quant_mxfp4(x.to(DEV), act)
    xv = f32(x).astype(np.float64)
    a = orc.activation(xv[:, :d], act) * xv[:, d:]
    byte = mxfp4_row_scales(scale, d).cpu().numpy()
    got = orc.values(orc.unpack(codes.cpu().numpy()), byte)[:, :d]
    # the scale: from an amax within a bf16 rounding (2^-8) of the exact one
    B = orc.blocks(d)
    pad = np.zeros((M, B * 32))
    pad[:, :d] = np.abs(a)
    amax = pad.reshape(M, B, 32).max(2)
    lo, hi = np.floor(np.log2(np.maximum(amax * (1 - 2.0**-7), 2.0**-120))), np.floor(np.log2(np.maximum(amax * (1 + 2.0**-7), 2.0**-120)))
    e = byte.astype(int) - 127 + 2
    assert ((e >= lo) & (e <= hi) | (amax < 2.0**-119)).all()
    s = np.repeat(np.exp2(byte.astype(np.float64) - 127), 32, axis=1)[:, :d]
    q = np.abs(a) / s
    half = np.where(q < 2.05, 0.25, np.where(q < 4.1, 0.5, 1.0))
    sat = q > 6  # saturated (amax below 8)
    tol = half * s + np.abs(a) * (2.0**-8 + 2.0**-18)
    tol = np.where(sat, np.abs(a) - 6 * s + np.abs(a) * 2.0**-7, tol)
    assert (np.abs(got - a) <= tol).all()
    assert (orc.unpack(codes.cpu().numpy())[:, d:] == 0).all()


@pytest.mark.parametrize("M,H", [(1, 8), (3, 40), (1, 5120), (7, 520), (33, 1032), (130, 768), (2, 17408), (1, 32768),
                                 (2080, 1280), (5000, 2048), (600, 5120)])
@pytest.mark.parametrize("with_res", [False, True])
def test_rmsnorm_quant_equals_norm_then_quant(M, H, with_res):
    """One kernel gives y, the residual and the codes of the two it replaces."""
    announce(f"rmsnorm_quant_mxfp4 M={M} H={H} res={with_res}")
    gen = torch.Generator().manual_seed(M + H)
    x = _acts(M, H, seed=H).to(DEV)
    res = torch.randn(M, H, generator=gen).bfloat16().to(DEV) if with_res else None
    w = (torch.rand(H, generator=gen) * 1.5 + 0.25).bfloat16().to(DEV)
    r1 = res.clone() if with_res else None
    codes, scale, y = rmsnorm_quant_mxfp4(x, w, 1e-6, residual=r1, return_y=True)
    r2 = res.clone() if with_res else None
    want = rmsnorm_quant(x, w, 1e-6, residual=r2, quantize=False)
    assert torch.equal(y, want)
    if with_res:
        assert torch.equal(r1, r2)
    c2, s2 = quant_mxfp4(want)
    assert torch.equal(codes, c2) and torch.equal(scale, s2)
    c3, s3 = rmsnorm_quant_mxfp4(x, w, 1e-6, residual=res)[:2]
    assert torch.equal(codes, c3) and torch.equal(scale, s3)


def test_rmsnorm_quant_in_place_and_nan():
    announce("rmsnorm_quant_mxfp4 in place, NaN row")
    x = _acts(5, 1024, seed=2).to(DEV)
    x[1, 3] = float("nan")
    x[2] = 0
    w = torch.ones(1024, dtype=torch.bfloat16, device=DEV)
    want = rmsnorm_quant(x.clone(), w, 1e-6, quantize=False)
    codes, scale, y = rmsnorm_quant_mxfp4(x, w, 1e-6, y=x)
    assert y.data_ptr() == x.data_ptr() and torch.equal(y[0], want[0]) and torch.isnan(y[1]).all()
    rows = mxfp4_row_scales(scale, 1024)
    assert (rows[1] == 255).all() and (rows[2] == 0).all() and (rows[0] < 255).all()


def test_rmsnorm_quant_refuses_y_on_residual():
    """Both are written: the sum and the normalized row."""
    x, r = (torch.ones(4, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    with pytest.raises(ValueError, match="residual"):
        rmsnorm_quant_mxfp4(x, x[0], 1e-6, residual=r, y=r)
    assert (r == 1).all()


def test_empty_and_refusals():
    x = torch.zeros(0, 64, dtype=torch.bfloat16, device=DEV)
    codes, scale = quant_mxfp4(x)
    assert codes.shape == (0, 32) and scale.shape == (1, 0, 16)
    assert dequant_mxfp4(codes, scale).shape == (0, 64)
    y = torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV)
    for bad in (y.float(), y[0], y.t(), y.as_strided((3, 64), (16, 1))):
        with pytest.raises(ValueError):
            quant_mxfp4(bad)
    with pytest.raises(ValueError):
        act_and_mul_quant_mxfp4(y, "relu")
    with pytest.raises(ValueError):
        rmsnorm_quant_mxfp4(y, y[0], 1e-6, residual=y)
    c, s = quant_mxfp4(y)
    with pytest.raises(ValueError):
        dequant_mxfp4(c, s, 65)
    with pytest.raises(ValueError):
        dequant_mxfp4(c, s.cpu())
