"""CPU tests of the float weights that MXFP4 layers take: their bf16 stand-ins
quantize to the weights' own codes and scales."""

import numpy as np
import pytest
import torch

from minisgl_amd.layers.mxfp4 import _bf16_with_codes_of
from oracle import mxfp4 as orc

DTYPES = [torch.bfloat16, torch.float16, torch.float32, torch.float64]


def weights(dtype, seed=0):
    """Rows of 64: random ones over the exponents of the type, and the levels'
    midpoints (at many scales) with their neighbours in the type."""
    rng = np.random.default_rng(seed)
    info = torch.finfo(dtype)
    low, high = max(int(np.log2(info.smallest_normal)), -140), min(int(np.log2(info.max)), 127) - 4  # fp32's range
    rows = [torch.from_numpy(rng.standard_normal((40, 64)) * np.exp2(rng.integers(low, high, (40, 1)))).to(dtype)]
    for e in (low, low + 3, -10, -3, 0, 5, high - 3):
        mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64) * 2.0**e
        mid = mid.to(dtype)
        near = torch.cat([mid, torch.nextafter(mid, mid * 0), torch.nextafter(mid, mid * 2)]) if dtype != torch.bfloat16 else mid
        row = torch.zeros(64, dtype=dtype)
        row[: len(near)] = near
        row[32 : 32 + len(near)] = -near
        row[31] = row[63] = 4.0 * 2.0**e  # the block's scale is 2^e
        rows.append(row[None])
    return torch.cat(rows)


@pytest.mark.parametrize("dtype", DTYPES)
def test_stand_ins_have_the_codes(dtype):
    w = weights(dtype)
    got = orc.quantize(_bf16_with_codes_of(w).double().numpy())
    want = orc.quantize(w.double().numpy())
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(got[0], want[0])


def test_a_rounded_weight_would_not():
    """1.25 + 2^-20 lies above the midpoint of 1 and 1.5."""
    w = torch.zeros(1, 32)
    w[0, 0], w[0, 1] = 4.0, 1.25 + 2.0**-20
    assert orc.quantize(w.double().numpy())[0][0, 1] == 3
    assert orc.quantize(w.bfloat16().double().numpy())[0][0, 1] == 2
    assert orc.quantize(_bf16_with_codes_of(w).double().numpy())[0][0, 1] == 3


@pytest.mark.parametrize("dtype", DTYPES[2:])
def test_limits(dtype):
    w = torch.tensor([[float("nan"), float("inf"), float("-inf"), 0.0, -0.0, 3.4028234e38, 1e-45, -1e-45]], dtype=dtype)
    v = _bf16_with_codes_of(w)[0]
    assert torch.isnan(v[0]) and v[1] == float("inf") and v[2] == float("-inf")
    assert v[3] == 0 and v[4] == 0 and torch.signbit(v[4]) and torch.isfinite(v[5])
    assert 0 < v[6] < 2.0**-130 and -(2.0**-130) < v[7] < 0
    # a NaN whose payload lies in the dropped bits
    bits = torch.tensor([[0x7F800001]], dtype=torch.int32).view(torch.float32)
    assert torch.isnan(_bf16_with_codes_of(bits)).all()
    assert torch.isinf(_bf16_with_codes_of(torch.tensor([[1e300]], dtype=torch.float64))).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_takes_the_weights_codes(dtype):
    from minisgl_amd.layers import LinearMXFP4

    w = weights(dtype, seed=1)
    layer = LinearMXFP4(64, w.shape[0])
    layer.load_float_weight(w.to("cuda:0"))
    code, byte = orc.quantize(w.double().numpy())
    np.testing.assert_array_equal(layer.weight.cpu().numpy(), orc.pack(code))
    np.testing.assert_array_equal(layer.weight_scale.cpu().numpy(), orc.tile_scales(byte))
    layer.load_float_weight(w.t().contiguous().t().to("cuda:0"))
    np.testing.assert_array_equal(layer.weight.cpu().numpy(), orc.pack(code))
