"""The MXFP4 rings whose blocks walk over several output tiles, with the next
tile's loads in flight behind the stores of the one before: two to four tiles
per block, ragged last rows and columns, every store form, with and without
bias, a staggered start, the fused activation.

Inputs are exact (scales 1 and 2: every product is a multiple of 1/4 and sums
stay below 144 K < 2^22), so each result is the bits of the 64 x 64 tiling, whose
blocks own one tile, and of the fp64 product in some rows."""

import numpy as np
import pytest
import torch

from helpers import announce, f32
from minisgl_amd.kernel import act_and_mul_quant_mxfp4, gemm_act_mxfp4, gemm_mxfp4, load, mxfp4_tile_scales
from oracle import mxfp4 as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ONE_TILE = 4  # the tiling of 64 x 64


@pytest.fixture
def tuning():
    lib = load()
    yield lib.mw8_set_mxfp4_tuning
    lib.mw8_set_mxfp4_tuning(-1, 0)


def _operand(rows, K, seed, low=127):
    gen = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (rows, orc.blocks(K) * 16), dtype=torch.uint8, generator=gen)
    codes[:, K // 2 :] = 0
    byte = torch.randint(low, low + 2, (rows, orc.blocks(K)), dtype=torch.uint8, generator=gen)
    return (codes.to(DEV), mxfp4_tile_scales(byte.to(DEV))), (codes, byte)


def _values(host, rows):
    return orc.values(orc.unpack(host[0][rows].numpy()), host[1][rows].numpy())


@pytest.mark.parametrize("M,N,K", [(5100, 8200, 1504), (5100, 8196, 2080), (5100, 8197, 1056), (5000, 8193, 1600)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("cfg", [0, 1, 2])
def test_walk(tuning, cfg, bias, M, N, K):
    announce(f"gemm_mxfp4 walk cfg={cfg} M={M} N={N} K={K} bias={bias}")
    (a, ah), (w, wh) = _operand(M, K, seed=M + K), _operand(N, K, seed=N)
    b = torch.randint(-8, 9, (N,), generator=torch.Generator().manual_seed(N)) / 4 if bias else None
    bd = None if b is None else b.bfloat16().to(DEV)
    a[1][0, M // 3, 2] = 255  # a NaN row of the first tiles
    tuning(ONE_TILE, 0)
    want = gemm_mxfp4(*a, *w, bd)
    tuning(cfg, 0)
    buf = torch.full((M + 256, N), 3.0, dtype=torch.bfloat16, device=DEV)
    got = gemm_mxfp4(*a, *w, bd, out=buf[:M])
    assert torch.isnan(got[M // 3]).all() and torch.isnan(want[M // 3]).all()
    got[M // 3], want[M // 3] = 0, 0
    assert torch.equal(got, want) and (buf[M:] == 3).all()
    rows = [0, 1, 255, 256, M // 2, M - 2, M - 1]
    exact = orc.product(_values(ah, rows), _values(wh, slice(None)), None if b is None else b.double().numpy())[0]
    np.testing.assert_array_equal(f32(got[rows]).astype(np.float64), orc.round_bf16(exact))


@pytest.mark.parametrize("M,N,K,bias", [(4096, 34816, 4096, False), (4090, 34820, 3616, True), (4096, 34817, 4000, True)])
def test_staggered_walk(tuning, M, N, K, bias):
    """Eight tiles and more per block, at K past 3584."""
    announce(f"gemm_mxfp4 staggered walk M={M} N={N} K={K} bias={bias}")
    (a, _), (w, _) = _operand(M, K, seed=1), _operand(N, K, seed=2)
    b = (torch.randint(-8, 9, (N,), generator=torch.Generator().manual_seed(3)) / 4).bfloat16().to(DEV) if bias else None
    tuning(ONE_TILE, 0)
    want = gemm_mxfp4(*a, *w, b)
    tuning(0, 0)
    for _ in range(2):
        assert torch.equal(gemm_mxfp4(*a, *w, b), want)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,I,K", [(5000, 2048, 1504), (5100, 4128, 2080), (2100, 9760, 576)])
def test_activation_walk(tuning, act, M, I, K):
    announce(f"gemm_act_mxfp4 walk M={M} I={I} K={K} {act}")
    (a, _), (w, _) = _operand(M, K, seed=M), _operand(2 * I, K, seed=I, low=118)
    a[1][0, M // 3, 2] = 255
    tuning(ONE_TILE, 0)
    want = act_and_mul_quant_mxfp4(gemm_mxfp4(*a, *w), act)
    got = gemm_act_mxfp4(*a, *w, act)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("M", [2080, 4100])
def test_walk_in_a_graph(M):
    """Captured and replayed with new rows between eager products."""
    announce(f"gemm_mxfp4 walk in a graph M={M}")
    N, K = 17408, 1024
    (w, _), xs = _operand(N, K, seed=1), [_operand(M, K, seed=2 + i)[0] for i in range(2)]
    want = [gemm_mxfp4(*x, *w) for x in xs]
    q, s = xs[0][0].clone(), xs[0][1].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gemm_mxfp4(q, s, *w)
    for i in (1, 0, 1):
        q.copy_(xs[i][0]), s.copy_(xs[i][1])
        graph.replay()
        eager = gemm_mxfp4(*xs[1 - i], *w)
        torch.cuda.synchronize()
        assert torch.equal(y, want[i]) and torch.equal(eager, want[1 - i])
