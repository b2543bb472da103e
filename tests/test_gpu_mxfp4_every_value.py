"""The MXFP4 quantizer's conversion over its whole domain: every finite bf16
value under every block scale that a block holding it can have."""

import numpy as np
import pytest
import torch

from helpers import announce, f32
from minisgl_amd.kernel import mxfp4_row_scales, quant_mxfp4
from oracle import mxfp4 as orc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("low", range(0, 255, 51))
def test_every_value_under_every_scale(low):
    """For each binade of the block's maximum (biased exponents low .. low +
    50): blocks of the binade's largest value and 31 values not above it."""
    announce(f"quant_mxfp4 every value, exponents from {low}")
    rows = []
    for exponent in range(low, low + 51):
        most = (exponent << 7) | 0x7F
        mag = np.arange(most + 1, dtype=np.int32)
        v = np.concatenate([mag, mag | 0x8000])
        v = np.resize(v, (-(-len(v) // 31), 31))
        rows.append(np.concatenate([np.full((len(v), 1), most, np.int32), v], 1))
    x = torch.from_numpy(np.concatenate(rows).astype(np.uint16).view(np.int16)).view(torch.bfloat16)
    codes, scale = quant_mxfp4(x.to("cuda:0"))
    code, byte = orc.quantize(f32(x).astype(np.float64))
    assert len(np.unique(byte)) >= 49
    np.testing.assert_array_equal(mxfp4_row_scales(scale, 32).cpu().numpy(), byte)
    np.testing.assert_array_equal(codes.cpu().numpy(), orc.pack(code))
