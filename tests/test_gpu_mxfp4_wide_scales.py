"""GPU parity of the fused gate_up product, activation and quantizer, and of its
parts, where fp32 sums are not exact: block scales over 30 binades, so that the
order of additions matters and the kernels that the parts may run on differ.

Both stay within the bounds of the fp64 oracle.  A gate or up sum of K terms of
magnitudes summing to S is off by (K + 1) 2^-23 S, its bf16 rounding by 2^-8:
dg, du.  |act'| < 1.13, so h = act(g) u is off by dh = 1.13 dg (|u| + du) +
|act(g)| du + 2^-8 |h| (its own bf16 rounding) + (g^2 + 19) 2^-23 |h| for |g| up to
12 (the activation's steps; past it the activation is g, or below 2^-100 of the
block, and has none).  A block's scale comes from an amax within the largest
dh of the block, a code from a value within dh: half a spacing more, or what
saturates at 6."""

import numpy as np
import pytest
import torch

from helpers import announce
from minisgl_amd.kernel import act_and_mul_quant_mxfp4, gated_mlp_quantized_mxfp4, gemm_act_mxfp4, gemm_mxfp4, load, mxfp4_row_scales
from minisgl_amd.kernel import mxfp4_tile_scales
from oracle import mxfp4 as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _operand(rows, K, seed, low, high):
    rng = np.random.default_rng(seed)
    code = rng.integers(0, 16, (rows, orc.blocks(K) * 32)).astype(np.uint8)
    code[:, K:] = 0
    byte = rng.integers(low, high + 1, (rows, orc.blocks(K))).astype(np.uint8)
    dev = (torch.from_numpy(orc.pack(code)).to(DEV), mxfp4_tile_scales(torch.from_numpy(byte)).to(DEV))
    return dev, orc.values(code, byte)


def _within(got, av, wv, act, K):
    """(codes, scale) [M, I] against the oracle's act(gate) * up."""
    y, size = orc.product(av, wv)
    inter = wv.shape[0] // 2
    err = 2.0**-8 * np.abs(y) + (K + 1) * 2.0**-23 * size * (1 + 2.0**-8)
    g, u, dg, du = y[:, :inter], y[:, inter:], err[:, :inter], err[:, inter:]
    a = orc.activation(g, act)
    h = a * u
    dh = 1.13 * dg * (np.abs(u) + du) + np.abs(a) * du
    dh += (np.abs(h) + dh) * (2.0**-8 + (np.minimum(np.abs(g), 12) ** 2 + 19) * 2.0**-23) + 2.0**-126
    byte = mxfp4_row_scales(got[1], inter).cpu().numpy()
    e = byte.astype(int) - 127 + 2
    blocks = (len(h), -1, 32)
    amax, slack = np.abs(h).reshape(blocks).max(2), dh.reshape(blocks).max(2)
    low = np.floor(np.log2(np.maximum(amax - slack, 2.0**-125)))
    assert ((e >= low) & (e <= np.floor(np.log2(amax + slack)))).all()
    v = orc.values(orc.unpack(got[0].cpu().numpy()), byte)
    s = np.repeat(np.exp2(byte.astype(np.float64) - 127), 32, axis=1)
    most = (np.abs(h) + dh) / s
    half = np.where(most < 2, 0.25, np.where(most < 4, 0.5, np.maximum(1.0, most - 6)))
    assert (np.abs(v - h) <= half * s + dh).all()


SHAPES = [(20, 12320, 512), (8, 96, 1024), (64, 96, 17408), (40, 608, 5120), (300, 288, 2048), (3, 544, 1056)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,I,K", SHAPES)
def test_fused_and_parts(M, I, K, act):
    announce(f"gemm_act_mxfp4 wide scales M={M} I={I} K={K} {act}")
    a, av = _operand(M, K, seed=M + K, low=112, high=142)
    w, wv = _operand(2 * I, K, seed=I, low=82, high=112)
    _within(gemm_act_mxfp4(*a, *w, act), av, wv, act, K)
    _within(act_and_mul_quant_mxfp4(gemm_mxfp4(*a, *w), act), av, wv, act, K)


@pytest.mark.parametrize("M,I,K", [(20, 32768, 5120), (300, 1056, 1024)])
def test_mlp_is_its_parts(M, I, K):
    """The MLP runs gate_up as gemm_act_mxfp4 or as product and activation, by
    what the library prefers, then the product: their bits."""
    announce(f"gated_mlp_mxfp4 wide scales M={M} I={I} K={K}")
    gen = torch.Generator().manual_seed(M)

    def operand(rows, k):
        codes = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, generator=gen)
        scale = torch.randint(96, 127, (rows, k // 32), dtype=torch.uint8, generator=gen)
        return codes.to(DEV), mxfp4_tile_scales(scale.to(DEV))

    a, w1, w2 = operand(M, K), operand(2 * I, K), operand(256, I)
    if load().mw8_gemm_act_mxfp4_preferred(M, I, K):
        h = gemm_act_mxfp4(*a, *w1)
    else:
        h = act_and_mul_quant_mxfp4(gemm_mxfp4(*a, *w1))
    assert torch.equal(gated_mlp_quantized_mxfp4(*a, *w1, *w2), gemm_mxfp4(*h, *w2))
