"""CPU tests of the MXFP4 products' choices (256 compute units without a GPU)."""

import pytest

from minisgl_amd.kernel import load


@pytest.mark.parametrize("M", [17, 24, 32])
@pytest.mark.parametrize("I,K", [(32768, 5120), (65536, 5120), (32768, 6144), (16384, 5120)])
def test_no_fused_activation_where_a_decode_kernel_runs(M, I, K):
    """Up to 32 rows on many weight rows the product streams its weights once,
    faster than 256-row tiles of which one in eight rows is filled."""
    assert load().mw8_gemm_act_mxfp4_preferred(M, I, K) == 0


def test_fused_activation_of_larger_batches():
    lib = load()
    for M, I, K in ((200, 25600, 5120), (2080, 25600, 5120), (2080, 17408, 5120), (1024, 6400, 5120), (8192, 768, 2048),
                    (64, 32768, 5120)):
        assert lib.mw8_gemm_act_mxfp4_preferred(M, I, K) == 1
    for M, I, K in ((16, 65536, 5120), (333, 17408, 5120), (1024, 768, 2048)):
        assert lib.mw8_gemm_act_mxfp4_preferred(M, I, K) == 0


def test_rows_of_the_one_launch_linear():
    """A wave quantizes its tiles of every row in 8 passes, 4 in single row groups."""
    takes = load().mw8_linear_bf16_mxfp4_supported
    assert [m for m in range(1, 17) if takes(m, 512, 512)] == list(range(1, 9))
    assert [m for m in range(1, 17) if takes(m, 7168, 5120)] == [1, 2]
    for n in (16, 8192, 8193, 60000):
        for k in (32, 512, 2048, 5120, 17408, 1 << 20):
            assert not any(takes(m, n, k) for m in range(9, 17))
