"""CPU tests of the rotary operators: refusals before any launch."""

import ctypes

import pytest
import torch

from minisgl_amd.kernel import load, rotary_cos_sin, rotary_qk


def test_c_refusals():
    lib = load()
    ARG, SHAPE, ALIGN = 1, 2, 3
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4098)

    def call(q=p, hq=2, k=p, hk=1, dtype=0, D=64, R=64, pos=p, pos64=1, table=p, P=8, eps=1e-6, T=4):
        return lib.mw8_rotary_qk(q, 128, 64, hq, k, 64, 64, hk, q, 128, 64, k, 64, 64, dtype, D, R, 0, pos, pos64, table, P,
                                 None, None, eps, T, None)

    assert call(T=0) == 0
    assert call(q=None) == ARG and call(k=None) == ARG and call(pos=None) == ARG and call(table=None) == ARG
    assert call(dtype=3) == ARG and call(dtype=-1) == ARG and call(eps=-1.0) == ARG and call(eps=float("nan")) == ARG
    assert call(T=-1) == SHAPE and call(hq=-1) == SHAPE and call(hq=0, hk=0) == SHAPE
    assert call(R=0) == SHAPE and call(R=63) == SHAPE and call(R=66) == SHAPE and call(D=0) == SHAPE and call(D=8194) == SHAPE
    assert call(P=0) == SHAPE and call(T=1 << 31) == SHAPE and call(hq=1 << 20, T=1 << 12) == SHAPE
    assert call(dtype=2, q=odd) == ALIGN and call(pos=odd) == ALIGN and call(table=odd) == ALIGN
    assert lib.mw8_rotary_cos_sin(None, 4, 8, 1.0, p, None) == ARG
    assert lib.mw8_rotary_cos_sin(p, 0, 8, 1.0, p, None) == SHAPE
    assert lib.mw8_rotary_cos_sin(p, 4, -1, 1.0, p, None) == SHAPE
    assert lib.mw8_rotary_cos_sin(odd, 4, 8, 1.0, p, None) == ALIGN
    assert lib.mw8_rotary_cos_sin(p, 4, 0, 1.0, p, None) == 0


def test_c_refuses_many_heads_and_odd_weights():
    lib = load()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4097)

    def call(hq, hk, qw, kw):
        return lib.mw8_rotary_qk(p, 128, 64, hq, p, 64, 64, hk, p, 128, 64, p, 64, 64, 0, 64, 64, 0, p, 1, p, 8, qw, kw, 1e-6, 4,
                                 None)

    for hq, hk in ((2**31 - 1, 1), (1, 2**31 - 1), (2**31 - 1, 2**31 - 1)):
        assert call(hq, hk, None, None) == 2
    assert call(2, 1, odd, None) == 3 and call(2, 1, None, odd) == 3


def test_python_refuses_cpu_tensors():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        rotary_qk(q, q, torch.arange(4), torch.zeros(8, 64))
    with pytest.raises(ValueError):
        rotary_cos_sin(torch.ones(4, dtype=torch.float64), 8)
