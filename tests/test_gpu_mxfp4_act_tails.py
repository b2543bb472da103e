"""GPU parity of the MXFP4 gated activation where it is small: blocks of 32
whose gates all lie in the activation's tail, so that the block's own scale
magnifies the activation's relative error.

Tolerances, in fp32 steps of 2^-23 relative: gelu's tail is a e^(-g^2 / 2) h(a), a =
|g|.  g^2 is exact, the exponent's constant and product are off by 1/2 each, which
moves e^(-g^2 / 2) by g^2 / 2 at most; the exponential itself 1, the reciprocal and its
argument 1.5 (h grows no faster than the reciprocal), the polynomial 1.2 with its
fit and 1/2 for each of 7 steps on partial sums of at most 1.5 times the result, three
products 1.5, the product with up 1/2: delta = (g^2 + 19) 2^-23 is more than that.
silu's e^-g has an exponent |g| / ln 2 off by 2^-23 of itself, |g| steps of the
result; the exponential 1, the reciprocal and its argument 1.5, products 1: delta = (|g| + 8) 2^-23.
The bf16 rounding adds 2^-8, and half a spacing of the code the rest."""

import numpy as np
import pytest
import torch

from helpers import announce, f32
from minisgl_amd.kernel import act_and_mul_quant_mxfp4, gemm_act_mxfp4, gemm_mxfp4, mxfp4_row_scales, mxfp4_tile_scales
from oracle import mxfp4 as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _check(x, act, delta):
    """x bf16 [M, 2d], d % 32 == 0, nonzero activations: the quantizer's values
    lie within delta, the bf16 rounding and half a code's spacing of the exact
    ones, and its scales come from an amax as near."""
    d = x.shape[1] // 2
    codes, scale = act_and_mul_quant_mxfp4(x.to(DEV), act)
    xv = f32(x).astype(np.float64)
    a = orc.activation(xv[:, :d], act) * xv[:, d:]
    err = 2.0**-8 + delta
    byte = mxfp4_row_scales(scale, d).cpu().numpy()
    amax = np.abs(a).reshape(len(a), -1, 32).max(2)
    e = byte.astype(int) - 127 + 2
    wide = 1 + err.reshape(len(a), -1, 32).max(2)
    assert ((e >= np.floor(np.log2(amax / wide))) & (e <= np.floor(np.log2(amax * wide)))).all()
    got = orc.values(orc.unpack(codes.cpu().numpy()), byte)
    s = np.repeat(np.exp2(byte.astype(np.float64) - 127), 32, axis=1)
    q = np.abs(a) / s
    half = np.where(q < 2 * (1 + err), 0.25, np.where(q < 4 * (1 + err), 0.5, 1.0))
    tol = half * s + np.abs(a) * err
    tol = np.where(q > 6, np.maximum(np.abs(a) - 6 * s, s) + np.abs(a) * err, tol)  # saturated, amax below 8
    assert (np.abs(got - a) <= tol).all()


def _tail(low, high, seed):
    """Rows of 8 blocks, each block's gates one bf16 value of [low, high] (all of
    them in turn), its ups +-[1, 2)."""
    bits = torch.arange(32768, 65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)  # the negative values
    g = bits[(bits.float() >= low) & (bits.float() <= high)]
    g = g[torch.arange(-(-len(g) // 8) * 8) % len(g)]
    gen = torch.Generator().manual_seed(seed)
    u = (1 + torch.rand(len(g), 32, generator=gen)) * torch.where(torch.rand(len(g), 32, generator=gen) < 0.5, -1.0, 1.0)
    return torch.cat([g[:, None].expand(-1, 32).reshape(-1, 256), u.bfloat16().view(-1, 256)], 1)


def test_gelu_tail():
    announce("act_and_mul_quant_mxfp4 gelu tail")
    x = _tail(-12.5, -0.5, 1)
    _check(x, "gelu", (f32(x).astype(np.float64)[:, :256] ** 2 + 19) * 2.0**-23)


def test_silu_tail():
    """Down to where the reciprocal leaves fp32's normal range (2^-126, g = -87.3)."""
    announce("act_and_mul_quant_mxfp4 silu tail")
    x = _tail(-87.0, -0.5, 2)
    _check(x, "silu", (np.abs(f32(x).astype(np.float64)[:, :256]) + 8) * 2.0**-23)


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_zeros_keep_their_sign(act):
    """Gates of zero, and ones so low that the activation underflows, beside one
    that sets the block's scale: codes 0 and 8 by the oracle's signs."""
    announce(f"act_and_mul_quant_mxfp4 signed zeros {act}")
    gates = torch.tensor([1.0, 0.0, -0.0, -30.0, -200.0, -1e-40, 1e-40, -3e38] * 4)
    for up in (2.0, -2.0, 0.0, -0.0):
        x = torch.cat([gates, torch.full((32,), up)]).bfloat16()[None]
        codes, scale = act_and_mul_quant_mxfp4(x.to(DEV), act)
        xv = f32(x).astype(np.float64)
        code, byte = orc.quantize(orc.round_bf16(orc.activation(xv[:, :32], act) * xv[:, 32:]))
        np.testing.assert_array_equal(codes.cpu().numpy(), orc.pack(code))
        np.testing.assert_array_equal(mxfp4_row_scales(scale, 32).cpu().numpy(), byte)


def _rows_of_gates(count, value, N, seed):
    """Quantized A [M, 64] of ones in the first count[m] columns, zeros behind,
    and W [2 N, 64]: gate rows `value`, up rows random levels.  So the gates of
    row m are count[m] value, and every sum is exact."""
    code = np.where(np.arange(64)[None] < np.asarray(count)[:, None], 2, 0).astype(np.uint8)
    rng = np.random.default_rng(seed)
    w = np.full((2 * N, 64), int(np.argmin(np.abs(orc.LEVELS - abs(value)))) | (8 if value < 0 else 0), np.uint8)
    w[N:] = rng.integers(1, 8, (N, 64)) | 8 * rng.integers(0, 2, (N, 64))
    out = []
    for c in (code, w):
        byte = np.full((c.shape[0], 2), 127, np.uint8)
        out += [torch.from_numpy(orc.pack(c)).to(DEV), mxfp4_tile_scales(torch.from_numpy(byte)).to(DEV)]
    return out


@pytest.mark.parametrize("N", [64, 288])
def test_fused_gelu_tail_equals_its_parts(N):
    """The product's epilogue computes the same activation (exact sums)."""
    announce(f"gemm_act_mxfp4 gelu tail N={N}")
    ops = _rows_of_gates([m % 27 for m in range(300)], -0.5, N, seed=N)
    want = act_and_mul_quant_mxfp4(gemm_mxfp4(*ops), "gelu")
    got = gemm_act_mxfp4(*ops, "gelu")
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("N", [64, 288])
def test_fused_silu_tail_equals_its_parts(N):
    announce(f"gemm_act_mxfp4 silu tail N={N}")
    ops = _rows_of_gates([m % 30 for m in range(300)], -3.0, N, seed=N)
    want = act_and_mul_quant_mxfp4(gemm_mxfp4(*ops), "silu")
    got = gemm_act_mxfp4(*ops, "silu")
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
