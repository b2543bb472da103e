"""GPU parity of the MXFP4 products.  Two kinds of inputs:

* exact: scales 1 and 2, so every product is a multiple of 1/4 and every
  partial sum, in whatever order, fits fp32's 24 bits (asserted): the result
  is the exact sum rounded once to bf16, bit for bit;
* any scale: fp32 sums of K terms, each addition off by at most 2^-23 of the
  sum of the terms' magnitudes (S), so |y - exact| <= 2^-8 |exact| (the bf16
  rounding) + (K + 1) 2^-23 S."""

import numpy as np
import pytest
import torch

from helpers import announce, f32
from minisgl_amd.kernel import gated_mlp_mxfp4, gemm_mxfp4, linear_mxfp4, mxfp4_tile_scales, quant_mxfp4
from oracle import mxfp4 as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _operand(rows, K, seed, low=127, high=128):
    """Random codes and scale bytes in [low, high]: (device pair, fp64 values)."""
    rng = np.random.default_rng(seed)
    code = rng.integers(0, 16, (rows, orc.blocks(K) * 32)).astype(np.uint8)
    code[:, K:] = 0
    byte = rng.integers(low, high + 1, (rows, orc.blocks(K))).astype(np.uint8)
    dev = (torch.from_numpy(orc.pack(code)).to(DEV), mxfp4_tile_scales(torch.from_numpy(byte)).to(DEV))
    return dev, orc.values(code, byte)


SIZES = [(1, 16, 32), (1, 1, 32), (1, 5120, 5120), (2, 100, 64), (3, 7168, 1024), (5, 129, 160), (8, 512, 2080),
         (9, 640, 544), (15, 48, 512), (16, 1000, 5120), (17, 256, 1024), (31, 300, 992), (33, 129, 512), (48, 1024, 768),
         (64, 2048, 2048), (64, 5120, 1504), (65, 257, 1024), (100, 512, 3200), (127, 640, 256), (128, 768, 5120),
         (129, 384, 480), (200, 1000, 2048), (256, 256, 256), (257, 520, 1056), (333, 1111, 800), (512, 1024, 1024),
         (600, 264, 4096), (1025, 768, 288)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("bias", [False, True])
def test_gemm_exact(M, N, K, bias):
    announce(f"gemm_mxfp4 exact M={M} N={N} K={K} bias={bias}")
    a, av = _operand(M, K, seed=M + K)
    w, wv = _operand(N, K, seed=N * 3 + K)
    b = np.random.default_rng(N).integers(-8, 9, N) / 4 if bias else None
    y = gemm_mxfp4(*a, *w, None if b is None else torch.from_numpy(b).bfloat16().to(DEV))
    want, size = orc.product(av, wv, b)
    assert size.max() * 4 < 2**24
    np.testing.assert_array_equal(f32(y).astype(np.float64), orc.round_bf16(want))


@pytest.mark.parametrize("M,N,K", [(1, 7168, 5120), (7, 333, 1000), (16, 768, 2048), (40, 520, 17408), (130, 512, 5120),
                                   (300, 1000, 2048)])
def test_gemm_any_scale(M, N, K):
    announce(f"gemm_mxfp4 any scale M={M} N={N} K={K}")
    a, av = _operand(M, K, seed=1, low=110, high=140)
    w, wv = _operand(N, K, seed=2, low=100, high=130)
    y = f32(gemm_mxfp4(*a, *w)).astype(np.float64)
    want, size = orc.product(av, wv)
    assert (np.abs(y - want) <= 2.0**-8 * np.abs(want) + (K + 1) * 2.0**-23 * size).all()


@pytest.mark.parametrize("M", [1, 16, 50, 300])
def test_gemm_extreme_scales(M):
    """A NaN scale byte makes its row or column NaN and nothing else; the
    smallest and largest scales give zeros and infinities without NaN."""
    announce(f"gemm_mxfp4 extreme scales M={M}")
    N, K = 300, 1056
    a, av = _operand(M, K, seed=4)
    w, wv = _operand(N, K, seed=5)
    a[1][0, M // 2, 3] = 255
    w[1][1, 17, 9] = 255
    y = gemm_mxfp4(*a, *w)
    nan = torch.isnan(y)
    want = torch.zeros_like(nan)
    want[M // 2] = True
    want[:, 17] = True
    assert torch.equal(nan, want)
    a, av = _operand(M, K, seed=6, low=0, high=0)
    w, wv = _operand(N, K, seed=7, low=20, high=60)
    assert not gemm_mxfp4(*a, *w).float().abs().gt(1e-30).any()
    a, _ = _operand(M, K, seed=8, low=254, high=254)
    w, _ = _operand(N, K, seed=9, low=0, high=0)
    assert torch.isfinite(gemm_mxfp4(*a, *w).float()).all()


@pytest.mark.parametrize("M,K,N", [(1, 5120, 512), (1, 1000, 64), (4, 5120, 7168), (8, 2048, 768), (16, 5120, 640),
                                   (16, 999, 100), (17, 2048, 768), (100, 520, 264), (333, 5120, 512)])
@pytest.mark.parametrize("bias", [False, True])
def test_linear(M, K, N, bias):
    """Codes of x are exact, so the only error is the product's."""
    announce(f"linear_mxfp4 M={M} K={K} N={N} bias={bias}")
    gen = torch.Generator().manual_seed(M + N)
    x = torch.randn(M, K, generator=gen).bfloat16()
    b = torch.randn(N, generator=gen).bfloat16() if bias else None
    w, wv = _operand(N, K, seed=N, low=110, high=120)
    y = f32(linear_mxfp4(x.to(DEV), *w, None if b is None else b.to(DEV))).astype(np.float64)
    want, size = orc.product(orc.values(*orc.quantize(f32(x).astype(np.float64))), wv,
                             None if b is None else f32(b).astype(np.float64))
    assert (np.abs(y - want) <= 2.0**-8 * np.abs(want) + (K + 1) * 2.0**-23 * size).all()


@pytest.mark.parametrize("M", [1, 3, 16])
def test_linear_layouts(M):
    """Strided, misaligned and batched rows give the bits of the packed ones."""
    gen = torch.Generator().manual_seed(M)
    K, N = 1024, 320
    w, _ = _operand(N, K, seed=1)
    x = torch.randn(M, K, generator=gen).bfloat16().to(DEV)
    want = linear_mxfp4(x, *w)
    wide = torch.zeros(M, K + 24, dtype=torch.bfloat16, device=DEV)
    for off in (0, 8, 3):
        v = wide[:, off : off + K]
        v.copy_(x)
        assert torch.equal(linear_mxfp4(v, *w), want)
    assert torch.equal(linear_mxfp4(x.view(1, M, K), *w), want.view(1, M, N))
    assert torch.equal(linear_mxfp4(x.t().contiguous().t(), *w), want)
    assert torch.equal(linear_mxfp4(x[0], *w), want[0])
    assert torch.equal(gemm_mxfp4(*quant_mxfp4(x), *w), want)
    x[0, 5] = float("inf")
    y = linear_mxfp4(x, *w)
    assert torch.isnan(y[0]).all() and torch.equal(y[1:], want[1:])


@pytest.mark.parametrize("M", [1, 2])
def test_linear_of_rows_far_apart(M):
    """Last tokens of long sequences: rows 2^26 elements and more apart."""
    K, far = 512, (1 << 26) + 8
    announce(f"linear_mxfp4 M={M} rows {far} apart")
    w, _ = _operand(64, K, seed=1)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).bfloat16().to(DEV)
    store = torch.empty((M - 1) * far + K, dtype=torch.bfloat16, device=DEV)
    view = store.as_strided((M, K), (far, 1))
    view.copy_(x)
    assert torch.equal(linear_mxfp4(view, *w), linear_mxfp4(x, *w))


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,H,I", [(1, 512, 768), (5, 1000, 500), (16, 2048, 768), (70, 512, 640), (300, 1024, 1056),
                                   (1100, 512, 384)])
def test_gated_mlp(M, H, I, act):
    """The chain against itself in fp64.  gate and up are bf16 roundings of
    fp32 sums, so a sum near a rounding border may round the other way, move
    the activation by a bf16 step and a code by its spacing: such a code
    changes h by at most a third of its value (the widest spacing, 4 to 6,
    is a half of 4 and a third of 6; below 0.5 the value itself is under a
    quarter of the smallest nonzero level).  Sums of fp32 differ from
    fp64's by under 2^-20 of S, bf16 borders lie 2^-8 apart and codes change
    only within 2^-8 of theirs: fewer than 1 in 1000 codes.  The rms of the
    output moves by less than sqrt(1/1000) / 2 < 2%."""
    announce(f"gated_mlp_mxfp4 M={M} H={H} I={I} {act}")
    gen = torch.Generator().manual_seed(M + I)
    x = torch.randn(M, H, generator=gen).bfloat16()
    w1, v1 = _operand(2 * I, H, seed=1, low=118, high=121)
    w2, v2 = _operand(H, I, seed=2, low=118, high=121)
    y = f32(gated_mlp_mxfp4(x.to(DEV), *w1, *w2, act)).astype(np.float64)
    gu = orc.round_bf16(orc.product(orc.values(*orc.quantize(f32(x).astype(np.float64))), v1)[0])
    h = orc.round_bf16(orc.activation(gu[:, :I], act) * gu[:, I:])
    want = orc.product(orc.values(*orc.quantize(h)), v2)[0]
    assert np.linalg.norm(y - want) <= 0.02 * np.linalg.norm(want)
    assert np.isfinite(y).all()


def test_gemm_out_and_empty():
    a, _ = _operand(4, 512, seed=1)
    w, _ = _operand(40, 512, seed=2)
    out = torch.full((6, 40), 7.0, dtype=torch.bfloat16, device=DEV)
    y = gemm_mxfp4(*a, *w, out=out[:4])
    assert y.data_ptr() == out.data_ptr() and (out[4:] == 7).all()
    assert torch.equal(y, gemm_mxfp4(*a, *w))
    e = gemm_mxfp4(a[0][:0], a[1][:, :0].contiguous(), *w)
    assert e.shape == (0, 40)
    assert linear_mxfp4(torch.zeros(0, 512, dtype=torch.bfloat16, device=DEV), *w).shape == (0, 40)


def test_gemm_refusals():
    a, _ = _operand(4, 512, seed=1)
    w, _ = _operand(40, 512, seed=2)
    v, _ = _operand(40, 544, seed=2)
    bias = torch.zeros(40, dtype=torch.bfloat16, device=DEV)
    for call in (
        lambda: gemm_mxfp4(*a, *v),
        lambda: gemm_mxfp4(*a, w[0], v[1]),
        lambda: gemm_mxfp4(a[0].int(), a[1], *w),
        lambda: gemm_mxfp4(a[0][:, :16], a[1], *w),
        lambda: gemm_mxfp4(*a, *w, bias=bias.float()),
        lambda: gemm_mxfp4(*a, *w, bias=bias[:39]),
        lambda: gemm_mxfp4(*a, *w, bias=bias.cpu()),
        lambda: gemm_mxfp4(*a, *w, out=torch.zeros(4, 41, dtype=torch.bfloat16, device=DEV)),
        lambda: linear_mxfp4(torch.zeros(4, 480, dtype=torch.bfloat16, device=DEV), *w),
        lambda: linear_mxfp4(torch.zeros(4, 512, dtype=torch.float16, device=DEV), *w),
        lambda: gated_mlp_mxfp4(torch.zeros(4, 512, dtype=torch.bfloat16, device=DEV), *w, *w),
    ):
        with pytest.raises(ValueError):
            call()


def test_gemm_refuses_out_on_bias():
    a, _ = _operand(4, 512, seed=1)
    w, _ = _operand(40, 512, seed=2)
    out = torch.zeros(5, 40, dtype=torch.bfloat16, device=DEV)
    for bias in (out[0], out[3], out.view(-1)[150:190]):
        with pytest.raises(ValueError, match="overlap"):
            gemm_mxfp4(*a, *w, bias=bias, out=out[:4])
    gemm_mxfp4(*a, *w, bias=out[4], out=out[:4])


@pytest.mark.parametrize("M", [1, 16, 64, 200, 1100])
def test_streams_and_graph(M):
    """Eager on the current stream, on a side stream, and captured and replayed
    with new inputs between eager calls: the same bits."""
    announce(f"mxfp4 chain on streams and in a graph M={M}")
    gen = torch.Generator().manual_seed(M)
    H, I = 1024, 768
    w1, _ = _operand(2 * I, H, seed=1, low=118, high=121)
    w2, _ = _operand(H, I, seed=2, low=118, high=121)
    xs = [torch.randn(M, H, generator=gen).bfloat16().to(DEV) for _ in range(4)]
    want = [gated_mlp_mxfp4(x, *w1, *w2) for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [gated_mlp_mxfp4(x, *w1, *w2) for x in xs]
    side.synchronize()
    for g, r in zip(got, want):
        assert torch.equal(g, r)
    static = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gated_mlp_mxfp4(static, *w1, *w2)
    for i in (1, 2, 3, 0, 1):
        static.copy_(xs[i])
        graph.replay()
        eager = gated_mlp_mxfp4(xs[(i + 1) % 4], *w1, *w2)
        torch.cuda.synchronize()
        assert torch.equal(y, want[i]) and torch.equal(eager, want[(i + 1) % 4])


@pytest.fixture
def tuning():
    from minisgl_amd.kernel import load

    lib = load()
    yield lib.mw8_set_mxfp4_tuning
    lib.mw8_set_mxfp4_tuning(-1, 0)


@pytest.mark.parametrize("M,N,K", [(1, 16, 32), (17, 72, 544), (40, 1000, 1024), (130, 252, 2080), (300, 519, 288),
                                   (513, 1544, 1504), (1100, 1050, 992)])
@pytest.mark.parametrize("cfg", range(5))
def test_every_tiling(tuning, cfg, M, N, K):
    """Every tiling at every size, exact inputs: the automatic choice's bits."""
    from minisgl_amd.kernel import load

    assert load().mw8_mxfp4_tuning_count() == 5
    announce(f"gemm_mxfp4 tiling {cfg} M={M} N={N} K={K}")
    a, av = _operand(M, K, seed=M)
    w, wv = _operand(N, K, seed=N)
    b = np.random.default_rng(N).integers(-8, 9, N) / 4
    tuning(cfg, 0)
    want, size = orc.product(av, wv, b)
    assert size.max() * 4 < 2**24
    bias = torch.from_numpy(b).bfloat16().to(DEV)
    np.testing.assert_array_equal(f32(gemm_mxfp4(*a, *w, bias)).astype(np.float64), orc.round_bf16(want))
    # an output whose rows are not 16-byte aligned
    out = torch.empty(M * N + 1, dtype=torch.bfloat16, device=DEV)[1:].view(M, N)
    np.testing.assert_array_equal(f32(gemm_mxfp4(*a, *w, bias, out=out)).astype(np.float64), orc.round_bf16(want))


@pytest.mark.parametrize("M,N,K", [(17, 64, 1024), (64, 516, 17408), (100, 260, 4128), (65, 1032, 1536)])
@pytest.mark.parametrize("split", [2, 3, 5, 16])
def test_split(tuning, split, M, N, K):
    """K ranges through the workspace: the same bits on exact inputs, twice the
    same bits on any."""
    announce(f"gemm_mxfp4 split {split} M={M} N={N} K={K}")
    a, av = _operand(M, K, seed=M)
    w, wv = _operand(N, K, seed=N)
    b = np.random.default_rng(N).integers(-8, 9, N) / 4
    tuning(4, split)
    want, _ = orc.product(av, wv, b)
    y = gemm_mxfp4(*a, *w, torch.from_numpy(b).bfloat16().to(DEV))
    np.testing.assert_array_equal(f32(y).astype(np.float64), orc.round_bf16(want))
    a, _ = _operand(M, K, seed=1, low=100, high=150)
    assert torch.equal(gemm_mxfp4(*a, *w), gemm_mxfp4(*a, *w))


def test_workspace():
    """The size the library asks for, a workspace that is too small, and none."""
    from minisgl_amd.kernel import load
    from minisgl_amd.kernel.lib import MW8Error, check

    lib = load()
    M, N, K = 64, 5120, 17408
    need = lib.mw8_gemm_mxfp4_workspace_bytes(M, N, K)
    assert need > 0 and need % (M * N * 4) == 0
    assert lib.mw8_gemm_mxfp4_workspace_bytes(8192, 34816, 5120) == 0 and lib.mw8_gemm_mxfp4_workspace_bytes(1, N, K) == 0
    a, av = _operand(M, K, seed=1)
    w, wv = _operand(N, K, seed=2)
    want = gemm_mxfp4(*a, *w)
    y = torch.empty_like(want)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    st = torch.cuda.current_stream().cuda_stream
    args = (a[0].data_ptr(), a[1].data_ptr(), w[0].data_ptr(), w[1].data_ptr(), None, y.data_ptr(), M, N, K)
    with pytest.raises(MW8Error, match="WORKSPACE"):
        check(lib.mw8_gemm_mxfp4_bf16(*args, ws.data_ptr(), need - 1, st))
    check(lib.mw8_gemm_mxfp4_bf16(*args, ws.data_ptr(), need, st))
    assert torch.equal(y, want)
    y.zero_()
    check(lib.mw8_gemm_mxfp4_bf16(*args, None, 0, st))
    assert torch.equal(y, want)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,I,K", [(1, 32, 32), (3, 96, 544), (100, 160, 1024), (257, 128, 480), (300, 768, 2048),
                                   (700, 1504, 512), (2080, 544, 1024), (5000, 2048, 256)])
def test_gemm_act_equals_its_parts(act, M, I, K):
    """gate_up product, activation and quantizer in one launch: the codes and
    scale bytes of the three on exact inputs (any fp32 order gives the same
    sums), bytes past I included; a NaN reaches its row's blocks only."""
    from minisgl_amd.kernel import act_and_mul_quant_mxfp4, gemm_act_mxfp4

    announce(f"gemm_act_mxfp4 M={M} I={I} K={K} {act}")
    a, _ = _operand(M, K, seed=M)
    w, _ = _operand(2 * I, K, seed=I, low=118, high=119)
    a[1][0, M // 2, 0] = 255
    want = act_and_mul_quant_mxfp4(gemm_mxfp4(*a, *w), act)
    got = gemm_act_mxfp4(*a, *w, act)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_gemm_act_refusals():
    from minisgl_amd.kernel import gemm_act_mxfp4, load

    a, _ = _operand(4, 512, seed=1)
    for rows in (40, 66):
        w, _ = _operand(rows, 512, seed=2)
        with pytest.raises(ValueError):
            gemm_act_mxfp4(*a, *w)
    w, _ = _operand(64, 512, seed=2)
    with pytest.raises(ValueError):
        gemm_act_mxfp4(*a, *w, "relu")
    assert gemm_act_mxfp4(a[0][:0], a[1][:, :0].contiguous(), *w)[0].shape == (0, 16)
    lib = load()
    assert lib.mw8_gemm_act_mxfp4_supported(1, 32, 1) and not lib.mw8_gemm_act_mxfp4_supported(1, 33, 32)
    assert not lib.mw8_gemm_act_mxfp4_supported(1, 1 << 21, 1 << 11)


def test_two_streams_at_once():
    """Split products (fp32 sums in a workspace per call) queued on two streams
    without a wait between them: the bits of one after the other."""
    announce("split products on two streams")
    w, _ = _operand(1024, 17408, seed=1, low=118, high=121)
    a = [_operand(64, 17408, seed=2 + i, low=118, high=121)[0] for i in range(2)]
    want = [gemm_mxfp4(*x, *w) for x in a]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(gemm_mxfp4(*a[i], *w))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_other_threads_tuning_is_its_own():
    """A tiling override holds on its thread only."""
    import threading

    from minisgl_amd.kernel import load

    lib = load()
    sizes = []

    def other():
        lib.mw8_set_mxfp4_tuning(0, 0)
        sizes.append(lib.mw8_linear_bf16_mxfp4_supported(1, 512, 512))

    thread = threading.Thread(target=other)
    thread.start()
    thread.join()
    sizes.append(lib.mw8_linear_bf16_mxfp4_supported(1, 512, 512))
    assert sizes == [0, 1]


@pytest.mark.parametrize("M", [1, 16, 17, 64, 333])
def test_gemm_rows_behind_the_last(M):
    """An out that is the head of a larger buffer: the rows behind it stay."""
    announce(f"gemm_mxfp4 rows behind M={M}")
    for N in (520, 517):
        a, _ = _operand(M, 1024, seed=M)
        w, _ = _operand(N, 1024, seed=N)
        buf = torch.full((M + 300, N), 3.0, dtype=torch.bfloat16, device=DEV)
        y = gemm_mxfp4(*a, *w, out=buf[:M])
        assert torch.equal(y, gemm_mxfp4(*a, *w)) and (buf[M:] == 3).all()


MANY = 24576  # weight rows from which 8 to 32 tokens are kept on chip (256 compute units)


@pytest.mark.parametrize("M", [7, 8, 16, 17, 32, 33])
@pytest.mark.parametrize("N,K", [(MANY - 1, 32), (MANY, 32), (MANY + 1, 544), (MANY + 6, 1024), (MANY + 4, 500), (33000, 160)])
def test_many_weight_rows(M, N, K):
    """Few tokens on many weight rows, exact inputs; rows behind the last stay."""
    announce(f"gemm_mxfp4 many rows M={M} N={N} K={K}")
    a, av = _operand(M, K, seed=M)
    w, wv = _operand(N, K, seed=N)
    b = np.random.default_rng(N).integers(-8, 9, N) / 4
    bias = torch.from_numpy(b).bfloat16().to(DEV)
    buf = torch.full((M + 32, N), 3.0, dtype=torch.bfloat16, device=DEV)
    for bb, bd in ((None, None), (b, bias)):
        want, size = orc.product(av, wv, bb)
        assert size.max() * 4 < 2**24
        np.testing.assert_array_equal(f32(gemm_mxfp4(*a, *w, bd, out=buf[:M])).astype(np.float64), orc.round_bf16(want))
        assert (buf[M:] == 3).all()
    # an output whose rows are not 8-byte aligned
    odd = torch.empty(M * N + 1, dtype=torch.bfloat16, device=DEV)[1:].view(M, N)
    assert torch.equal(gemm_mxfp4(*a, *w, bias, out=odd), buf[:M])


@pytest.mark.parametrize("M", [9, 16, 31])
@pytest.mark.parametrize("N,K", [(34816, 5120), (51200, 5120), (40008, 6144), (40008, 6176), (70000, 1536)])
def test_many_weight_rows_equal_a_tiling(tuning, M, N, K):
    """Exact inputs (|sums| below 144 K < 2^22, multiples of 1/4): the bits of
    the tile rings."""
    announce(f"gemm_mxfp4 many rows M={M} N={N} K={K} against a tiling")
    gen = torch.Generator().manual_seed(M + N)
    ops = []
    for rows in (M, N):
        codes = torch.randint(0, 256, (rows, K // 2), dtype=torch.uint8, generator=gen)
        ops += [codes.to(DEV), mxfp4_tile_scales(torch.randint(127, 129, (rows, K // 32), dtype=torch.uint8, generator=gen)).to(DEV)]
    ops[1][0, M // 2, 3] = 255  # a NaN block reaches its row only
    got = gemm_mxfp4(*ops)
    tuning(2, 0)
    want = gemm_mxfp4(*ops)
    assert torch.isnan(want[M // 2]).all() and torch.isnan(got[M // 2]).all()
    keep = [m for m in range(M) if m != M // 2]
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("M", [16, 32])
def test_many_weight_rows_on_streams_and_in_a_graph(M):
    announce(f"gemm_mxfp4 many rows on streams and in a graph M={M}")
    w, _ = _operand(MANY, 1024, seed=1)
    xs = [_operand(M, 1024, seed=2 + i)[0] for i in range(3)]
    want = [gemm_mxfp4(*x, *w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(gemm_mxfp4(*xs[i % 3], *w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 3]) for i, y in enumerate(got))
    q, s = xs[0][0].clone(), xs[0][1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gemm_mxfp4(q, s, *w)
    for i in (1, 2, 0, 2):
        q.copy_(xs[i][0]), s.copy_(xs[i][1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i])


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,H,I,N", [(1, 512, 768, 512), (3, 1000, 500, 72), (8, 512, 12320, 264), (16, 2048, 768, 2048),
                                     (20, 512, 12320, 264), (64, 512, 4096, 512), (300, 1024, 1056, 1000), (2100, 512, 3200, 512)])
def test_gated_mlp_equals_its_parts(act, M, H, I, N):
    """One call, of rows as they lie and of quantized ones: the bits of
    quantizer, product, activation + quantizer and product."""
    from minisgl_amd.kernel import act_and_mul_quant_mxfp4, gated_mlp_quantized_mxfp4

    announce(f"gated_mlp_mxfp4 M={M} H={H} I={I} N={N} {act} against its parts")
    gen = torch.Generator().manual_seed(M + I)
    w1, _ = _operand(2 * I, H, seed=1, low=118, high=121)
    w2, _ = _operand(N, I, seed=2, low=118, high=121)
    wide = torch.randn(M, H + 8, generator=gen).bfloat16().to(DEV)
    for x in (wide[:, :H].contiguous(), wide[:, 8:], wide[:, 3 : H + 3]):
        q = quant_mxfp4(x)
        want = gemm_mxfp4(*act_and_mul_quant_mxfp4(linear_mxfp4(x, *w1), act), *w2)
        assert torch.equal(gated_mlp_mxfp4(x, *w1, *w2, act), want)
        if H % 32 == 0:
            want = gemm_mxfp4(*act_and_mul_quant_mxfp4(gemm_mxfp4(*q, *w1), act), *w2)
            assert torch.equal(gated_mlp_quantized_mxfp4(*q, *w1, *w2, act), want)


def test_gated_mlp_workspace():
    """The C entry stays inside the workspace it asks for, and refuses a
    smaller one."""
    from minisgl_amd.kernel import load
    from minisgl_amd.kernel.lib import check

    lib = load()
    announce("gated_mlp_mxfp4 workspace")
    w1, _ = _operand(2 * 4096, 512, seed=1, low=118, high=121)
    w2, _ = _operand(512, 4096, seed=2, low=118, high=121)
    for M in (1, 16, 64, 300, 2100):
        x = torch.randn(M, 512, generator=torch.Generator().manual_seed(M)).bfloat16().to(DEV)
        need = lib.mw8_gated_mlp_mxfp4_workspace_bytes(0, M, 512, 4096, 512)
        ws = torch.full((need + 4096,), 7, dtype=torch.uint8, device=DEV)
        y = torch.empty(M, 512, dtype=torch.bfloat16, device=DEV)
        args = (x.data_ptr(), 512, None, None, w1[0].data_ptr(), w1[1].data_ptr(), w2[0].data_ptr(), w2[1].data_ptr(), 0,
                y.data_ptr(), M, 512, 4096, 512, ws.data_ptr())
        st = torch.cuda.current_stream().cuda_stream
        assert lib.mw8_gated_mlp_mxfp4(*args, need - 1, st) != 0
        check(lib.mw8_gated_mlp_mxfp4(*args, need, st))
        assert (ws[need:] == 7).all() and torch.equal(y, gated_mlp_mxfp4(x, *w1, *w2))
