"""CPU tests of the MXFP4 operators: the oracle against the definition
element by element, the scale layout, and the refusals of the C entries and
of the Python wrappers (all before any launch)."""

import ctypes

import numpy as np
import pytest
import torch

from minisgl_amd.kernel import (
    act_and_mul_quant_mxfp4,
    dequant_mxfp4,
    gated_mlp_mxfp4,
    gemm_mxfp4,
    linear_mxfp4,
    load,
    mxfp4_row_scales,
    mxfp4_tile_scales,
    quant_mxfp4,
    rmsnorm_quant_mxfp4,
)
from oracle import mxfp4 as orc


def test_oracle_quantizer_is_the_definition():
    rng = np.random.default_rng(0)
    x = orc.round_bf16(rng.standard_normal((6, 75)) * np.exp2(rng.integers(-20, 20, (6, 75))))
    x[2] = 0
    x[3, :32] = 7.9  # saturates at 6 * 2^0
    code, byte = orc.quantize(x)
    assert code.shape == (6, 96) and byte.shape == (6, 3) and not code[:, 75:].any()
    for m in range(6):
        for b in range(3):
            blk = x[m, 32 * b : min(75, 32 * b + 32)]
            amax = np.abs(blk).max()
            e = max(int(np.floor(np.log2(amax))) - 2, -127) if amax > 0 else -127
            assert byte[m, b] == e + 127
            for i, v in enumerate(blk):
                assert code[m, 32 * b + i] & 7 == orc.nearest_level(abs(v) / 2.0**e)
    assert (orc.values(code, byte)[3, :32] == 6).all()


def test_oracle_ties_and_limits():
    x = np.array([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -5.0, -0.25] + [4.0] * 22])
    code, byte = orc.quantize(x)
    assert byte[0, 0] == 127
    np.testing.assert_array_equal(orc.values(code, byte)[0, :10], [0, 1, 1, 2, 2, 4, 4, 6, -4, 0])
    tiny = np.full((1, 32), 2.0**-133)
    code, byte = orc.quantize(tiny)
    assert byte[0, 0] == 0 and not code.any()
    for bad in (np.nan, np.inf, -np.inf):
        x[0, 5] = bad
        code, byte = orc.quantize(x)
        assert byte[0, 0] == 255 and not code.any() and np.isnan(orc.values(code, byte)).all()


@pytest.mark.parametrize("rows,k", [(1, 1), (3, 32), (5, 500), (4, 512), (2, 513), (7, 5120), (1, 1000)])
def test_scale_layout(rows, k):
    byte = np.random.default_rng(k).integers(0, 256, (rows, orc.blocks(k))).astype(np.uint8)
    t = mxfp4_tile_scales(torch.from_numpy(byte))
    np.testing.assert_array_equal(t.numpy(), orc.tile_scales(byte))
    np.testing.assert_array_equal(mxfp4_row_scales(t, k).numpy(), byte)


def test_round_bf16_matches_torch():
    rng = np.random.default_rng(3)
    x = (rng.standard_normal(20000) * np.exp2(rng.integers(-140, 127, 20000))).astype(np.float32)
    want = torch.from_numpy(x).bfloat16().float().numpy()
    np.testing.assert_array_equal(orc.round_bf16(x.astype(np.float64)).astype(np.float32), want)


def test_c_refusals():
    """Bad arguments return the documented code before anything is launched
    (the pointers are never read)."""
    lib = load()
    ARG, SHAPE, ALIGN = 1, 2, 3
    p = ctypes.c_void_p(4096)
    odd = ctypes.c_void_p(4097)
    assert lib.mw8_quant_mxfp4_bf16(None, 1, 32, 32, p, p, None) == ARG
    assert lib.mw8_quant_mxfp4_bf16(p, 1, 0, 32, p, p, None) == SHAPE
    assert lib.mw8_quant_mxfp4_bf16(p, -1, 32, 32, p, p, None) == SHAPE
    assert lib.mw8_quant_mxfp4_bf16(p, 1, 64, 32, p, p, None) == SHAPE
    assert lib.mw8_quant_mxfp4_bf16(p, 1 << 31, 32, 32, p, p, None) == SHAPE
    assert lib.mw8_quant_mxfp4_bf16(p, (1 << 31) - 1, 1 << 20, 1 << 20, p, p, None) == SHAPE
    assert lib.mw8_quant_mxfp4_bf16(odd, 1, 32, 32, p, p, None) == ALIGN
    assert lib.mw8_quant_mxfp4_bf16(p, 1, 32, 32, odd, p, None) == ALIGN
    assert lib.mw8_quant_mxfp4_bf16(p, 0, 32, 32, p, p, None) == 0
    assert lib.mw8_act_and_mul_quant_mxfp4_bf16(p, 1, 63, 0, p, p, None) == SHAPE
    assert lib.mw8_act_and_mul_quant_mxfp4_bf16(p, 1, 64, 2, p, p, None) == ARG
    assert lib.mw8_act_and_mul_quant_mxfp4_bf16(p, 1, 64, 0, p, None, None) == ARG
    assert lib.mw8_rmsnorm_quant_mxfp4_bf16(p, None, p, 1e-6, 1, 12, p, p, None, None) == SHAPE
    assert lib.mw8_rmsnorm_quant_mxfp4_bf16(p, None, p, 1e-6, 1, 32776, p, p, None, None) == SHAPE
    assert lib.mw8_rmsnorm_quant_mxfp4_bf16(p, None, p, -1.0, 1, 64, p, p, None, None) == ARG
    assert lib.mw8_rmsnorm_quant_mxfp4_bf16(p, None, p, 1e-6, 1, 64, None, p, p, None) == ARG
    assert lib.mw8_rmsnorm_quant_mxfp4_bf16(odd, None, p, 1e-6, 1, 64, p, p, None, None) == ALIGN
    assert lib.mw8_dequant_mxfp4_bf16(p, p, 1, 0, p, None) == SHAPE
    assert lib.mw8_dequant_mxfp4_bf16(p, None, 1, 32, p, None) == ARG
    assert lib.mw8_dequant_mxfp4_bf16(odd, p, 1, 32, p, None) == ALIGN
    assert lib.mw8_gemm_mxfp4_bf16(p, p, p, None, None, p, 1, 16, 32, None, 0, None) == ARG
    assert lib.mw8_gemm_mxfp4_bf16(p, p, p, p, None, p, 1, 0, 32, None, 0, None) == SHAPE
    assert lib.mw8_gemm_mxfp4_bf16(p, p, p, p, None, p, 1, 16, (1 << 20) + 1, None, 0, None) == SHAPE
    assert lib.mw8_gemm_mxfp4_bf16(p, p, odd, p, None, p, 1, 16, 32, None, 0, None) == ALIGN
    assert lib.mw8_gemm_mxfp4_bf16(p, p, p, p, None, p, 0, 16, 32, None, 0, None) == 0
    assert lib.mw8_last_error()


def test_fused_activation_limits():
    """256 rows of output codes must fit a 32-bit view: I / 2 * 256 < 2^31."""
    lib = load()
    p = ctypes.c_void_p(4096)
    assert lib.mw8_gemm_act_mxfp4_supported(256, (1 << 24) - 32, 32) == 1
    assert lib.mw8_gemm_act_mxfp4_supported(256, 1 << 24, 32) == 0
    assert lib.mw8_gemm_act_mxfp4(p, p, p, p, 0, p, p, 256, 1 << 24, 32, None) == 2


def test_launch_limits():
    """A launch holds fewer than 2^32 threads: one wave per row (or four rows)
    and 512 elements, four waves a block."""
    lib = load()
    p = ctypes.c_void_p(4096)
    rows = 1 << 26
    assert lib.mw8_dequant_mxfp4_bf16(p, p, rows, 32, p, None) == 2
    assert lib.mw8_dequant_mxfp4_bf16(p, p, rows // 8, 4096, p, None) == 2
    assert lib.mw8_quant_mxfp4_bf16(p, 4 * rows, 32, 32, p, p, None) == 2
    assert lib.mw8_act_and_mul_quant_mxfp4_bf16(p, 4 * rows, 64, 0, p, p, None) == 2


def test_gated_mlp_refusals():
    lib = load()
    p = ctypes.c_void_p(4096)

    def call(x=p, ldx=64, q=None, s=None, w=p, act=0, y=p, M=1, H=64, I=32, N=16, ws=p, ws_bytes=1 << 20):
        return lib.mw8_gated_mlp_mxfp4(x, ldx, q, s, w, p, p, p, act, y, M, H, I, N, ws, ws_bytes, None)

    assert call(M=0) == 0 and call(M=0, x=None, q=p, s=p) == 0
    assert call(x=None) == 1 and call(x=None, q=p) == 1 and call(w=None) == 1 and call(y=None) == 1 and call(act=2) == 1
    assert call(ldx=63) == 2 and call(H=0) == 2 and call(I=0) == 2 and call(N=0) == 2 and call(M=-1) == 2
    assert call(I=(1 << 20) + 1) == 2 and call(M=1 << 31) == 2
    need = lib.mw8_gated_mlp_mxfp4_workspace_bytes(0, 1, 64, 32, 16)
    assert need > 0 and call(ws_bytes=need - 1) == call(ws=None) != 0
    assert call(ws=ctypes.c_void_p(4100), ws_bytes=need) == 3
    assert lib.mw8_gated_mlp_mxfp4_workspace_bytes(0, 0, 64, 32, 16) == 0


def test_python_refuses_cpu_tensors():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    w, s = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(1, 8, 16, dtype=torch.uint8)
    for call in (
        lambda: quant_mxfp4(x),
        lambda: act_and_mul_quant_mxfp4(x),
        lambda: rmsnorm_quant_mxfp4(x, x[0], 1e-6),
        lambda: dequant_mxfp4(w, s),
        lambda: gemm_mxfp4(w, s, w, s),
        lambda: linear_mxfp4(x, w, s),
        lambda: gated_mlp_mxfp4(x, w, s, w, s),
    ):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):
        mxfp4_tile_scales(torch.zeros(2, 3))
    with pytest.raises(ValueError):
        mxfp4_row_scales(s, 1024)


def test_layers_state_and_refusals():
    from minisgl_amd.layers import GatedMLPMXFP4, LinearMXFP4, RMSNormQuantMXFP4

    layer = LinearMXFP4(1000, [64, 32], has_bias=True)
    assert layer.weight.shape == (96, 512) and layer.weight_scale.shape == (2, 96, 16) and layer.bias.shape == (96,)
    assert set(layer.state_dict()) == {"weight", "weight_scale", "bias"}
    codes = torch.zeros(96, 512, dtype=torch.uint8)
    rows = torch.randint(0, 255, (96, 32), dtype=torch.uint8)
    layer.load_mxfp4_weight(codes, rows, torch.ones(96))
    assert torch.equal(mxfp4_row_scales(layer.weight_scale, 1000), rows) and layer.bias.dtype == torch.bfloat16
    for bad in (
        lambda: layer.load_mxfp4_weight(codes[:, :500], rows),
        lambda: layer.load_mxfp4_weight(codes, rows[:, :31]),
        lambda: layer.load_mxfp4_weight(codes.int(), rows),
        lambda: layer.load_mxfp4_weight(codes, rows, torch.ones(95)),
        lambda: layer.load_float_weight(torch.zeros(96, 999)),
        lambda: layer.forward(torch.zeros(2, 1000, dtype=torch.bfloat16)),
        lambda: GatedMLPMXFP4(64, 64, "relu"),
    ):
        with pytest.raises(ValueError):
            bad()
    mlp = GatedMLPMXFP4(512, 256)
    assert mlp.gate_up_proj.output_size == 512 and mlp.down_proj.weight.shape == (512, 128)
    assert RMSNormQuantMXFP4(64, 1e-6).state_dict()["weight"].shape == (64,)
