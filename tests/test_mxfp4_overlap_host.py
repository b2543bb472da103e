"""CPU tests of the MXFP4 entries' overlap rules: an output that shares memory
with an input, another output or the workspace is refused before any launch
(the addresses are made up and never read)."""

import ctypes

import pytest

from minisgl_amd.kernel import load

ARG = 1
M, K, N = 64, 1024, 96
MB = 1 << 20


class At:
    """Addresses 1 MB apart, by name; `at` puts one at an offset from another."""

    def __init__(self, names, **moved):
        self.p = {n: (i + 1) * MB for i, n in enumerate(names)}
        for n, (other, off) in moved.items():
            self.p[n] = self.p[other] + off

    def __getitem__(self, n):
        return ctypes.c_void_p(self.p[n])


CODES, SCALES, Y = M * K // 2, K // 512 * M * 16, M * N * 2


@pytest.mark.parametrize("moved", [
    dict(q=("x", 0)), dict(q=("x", 2 * M * K - 4)), dict(q=("x", 4 - CODES)), dict(s=("x", 2 * K)), dict(s=("q", CODES - 4)),
    dict(s=("q", 4 - SCALES))])
def test_quantizers(moved):
    p = At("xqs", **moved)
    lib = load()
    assert lib.mw8_quant_mxfp4_bf16(p["x"], M, K, K, p["q"], p["s"], None) == ARG
    assert lib.mw8_act_and_mul_quant_mxfp4_bf16(p["x"], M, 2 * K, 0, p["q"], p["s"], None) == ARG


def test_quantizer_of_strided_rows():
    p = At("xqs", s=("x", 4 * 3 * K + 2 * K - 2))  # the end of row 3
    assert load().mw8_quant_mxfp4_bf16(p["x"], M, K, 2 * K, p["q"], p["s"], None) == ARG


@pytest.mark.parametrize("moved", [
    dict(r=("x", 0)), dict(r=("x", 2 * K)), dict(r=("x", -2 * K)), dict(y=("x", 2 * K)), dict(y=("r", 0)), dict(y=("r", -2 * K)),
    dict(w=("r", 2 * K * (M - 1))), dict(w=("y", 0)), dict(q=("x", 64)), dict(q=("y", 64)), dict(s=("r", 0)), dict(s=("q", 16))])
def test_norm(moved):
    p = At("xrwqsy", **moved)
    assert load().mw8_rmsnorm_quant_mxfp4_bf16(p["x"], p["r"], p["w"], 1e-6, M, K, p["q"], p["s"], p["y"], None) == ARG


@pytest.mark.parametrize("moved", [dict(y=("q", 0)), dict(y=("s", SCALES - 2)), dict(y=("q", 2 - 2 * M * K))])
def test_dequantizer(moved):
    p = At("qsy", **moved)
    assert load().mw8_dequant_mxfp4_bf16(p["q"], p["s"], M, K, p["y"], None) == ARG


@pytest.mark.parametrize("moved", [dict(y=("a", 0)), dict(y=("sa", 2 - Y)), dict(y=("w", N * K // 2 - 2)), dict(y=("sw", 0)),
                                   dict(y=("b", 2 - Y)), dict(b=("y", Y - 2))])
def test_product(moved):
    p = At(["a", "sa", "w", "sw", "b", "y"], **moved)
    lib = load()
    assert lib.mw8_gemm_mxfp4_bf16(p["a"], p["sa"], p["w"], p["sw"], p["b"], p["y"], M, N, K, None, 0, None) == ARG


@pytest.mark.parametrize("other", ["a", "sa", "w", "sw", "y"])
def test_product_workspace(other):
    lib = load()
    m, n, k = 64, 5120, 17408
    need = lib.mw8_gemm_mxfp4_workspace_bytes(m, n, k)
    assert need > 0
    p = {x: (i + 1) << 30 for i, x in enumerate(["a", "sa", "w", "sw", "y"])}
    ws = ctypes.c_void_p(p[other] + 16 - need)
    args = [ctypes.c_void_p(p[x]) for x in ("a", "sa", "w", "sw")]
    assert lib.mw8_gemm_mxfp4_bf16(*args, None, ctypes.c_void_p(p["y"]), m, n, k, ws, need, None) == ARG


@pytest.mark.parametrize("moved", [dict(y=("x", 0)), dict(y=("w", 2)), dict(y=("sw", 0)), dict(y=("b", 2 * N - 2))])
def test_linear(moved):
    p = At(["x", "w", "sw", "b", "y"], **moved)
    lib = load()
    assert lib.mw8_linear_bf16_mxfp4_supported(2, N, K)
    assert lib.mw8_linear_bf16_mxfp4(p["x"], K, p["w"], p["sw"], p["b"], p["y"], 2, N, K, None) == ARG


@pytest.mark.parametrize("moved", [dict(q=("a", 0)), dict(q=("sa", 8)), dict(q=("w", 8)), dict(s=("sw", 0)), dict(s=("q", 0))])
def test_product_with_activation(moved):
    p = At(["a", "sa", "w", "sw", "q", "s"], **moved)
    lib = load()
    assert lib.mw8_gemm_act_mxfp4(p["a"], p["sa"], p["w"], p["sw"], 0, p["q"], p["s"], M, N, K, None) == ARG


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("moved", [dict(y=("x", 0)), dict(y=("wg", 0)), dict(y=("sd", 0)), dict(ws=("x", 16)), dict(ws=("wd", 0)),
                                   dict(y=("ws", 512)), dict(ws=("sg", 0))])
def test_mlp(moved, quantized):
    p = At(["x", "s", "wg", "sg", "wd", "sd", "y", "ws"], **moved)
    lib = load()
    need = lib.mw8_gated_mlp_mxfp4_workspace_bytes(int(quantized), M, K, 64, N)
    rows = (None, 0, p["x"], p["s"]) if quantized else (p["x"], K, None, None)
    assert lib.mw8_gated_mlp_mxfp4(*rows, p["wg"], p["sg"], p["wd"], p["sd"], 0, p["y"], M, K, 64, N, p["ws"], need, None) == ARG


@pytest.mark.gpu
def test_refused_and_allowed_on_the_gpu():
    import torch

    from minisgl_amd.kernel import MW8Error, gemm_mxfp4, quant_mxfp4, rmsnorm_quant_mxfp4

    dev = "cuda:0"
    buf = torch.randn(6, 512, device=dev).bfloat16()
    keep, w = buf.clone(), torch.ones(512, dtype=torch.bfloat16, device=dev)
    for kw in (dict(residual=buf[1:5]), dict(y=buf[1:5])):
        with pytest.raises(MW8Error, match="overlap"):
            rmsnorm_quant_mxfp4(buf[:4], w, 1e-6, **kw)
    assert torch.equal(buf, keep)
    rmsnorm_quant_mxfp4(buf[:2], w, 1e-6, residual=buf[2:4], y=buf[4:])  # side by side
    # an output in the memory of an operand's codes
    mem = torch.zeros(64 * 256 * 2, dtype=torch.uint8, device=dev)
    codes, scale = quant_mxfp4(torch.randn(64, 512, device=dev).bfloat16())
    q = mem[: 64 * 256].view(64, 256)
    q.copy_(codes)
    wc, ws = quant_mxfp4(torch.randn(96, 512, device=dev).bfloat16())
    with pytest.raises(MW8Error, match="overlap"):
        gemm_mxfp4(q, scale, wc, ws, out=mem[: 64 * 96 * 2].view(torch.bfloat16).view(64, 96))
    out = mem[64 * 256 : 64 * 256 + 64 * 96 * 2].view(torch.bfloat16).view(64, 96)
    assert torch.equal(gemm_mxfp4(q, scale, wc, ws, out=out), gemm_mxfp4(codes, scale, wc, ws))
