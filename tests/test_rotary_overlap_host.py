"""CPU tests of the rotary operator's overlap rules: the row geometry against
marked bytes, and the C entry's refusals (before any launch; the pointers are
never read)."""

import ctypes
import os
import subprocess

import pytest

from minisgl_amd.kernel import load

ARG, SHAPE = 1, 2
D, SIZE = 64, 2


def test_row_geometry(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = tmp_path / "row_overlap_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", os.path.join(root, "mini-sglang-fork_amd", "csrc"),
                    os.path.join(root, "tests", "native", "row_overlap_check.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and "mismatches=0" in out.stdout, out.stdout + out.stderr


def call(q, k, q_out, k_out, T=4, hq=2, hk=1, pos=1 << 40, table=1 << 41, weight=None):
    """Each tensor an (element offset, token stride, head stride); addresses are
    made up, so only calls that are refused may be made."""
    def args(t):
        return ctypes.c_void_p((1 << 20) + SIZE * t[0]), t[1], t[2]

    return load().mw8_rotary_qk(*args(q), hq, *args(k), hk, *args(q_out), *args(k_out), 0, D, D, 0, ctypes.c_void_p(pos), 1,
                                ctypes.c_void_p(table), 8, None if weight is None else ctypes.c_void_p(weight), None, 1e-6, T, None)


LD = 256  # a qkv row of 2 + 1 + 1 heads
Q, K, V = (0, LD, D), (128, LD, D), (192, LD, D)
FAR = (1 << 20, LD, D)


@pytest.mark.parametrize("q,k,q_out,k_out", [
    (Q, K, (0, 128, D), K),                    # packed rows over the qkv rows that they come from
    (Q, K, (64, LD, D), (1 << 22, 64, D)),     # one head further
    (Q, K, (LD, LD, D), (1 << 22, 64, D)),     # one token further
    (Q, K, (0, LD, 2 * D), FAR),               # the same start, other head stride
    (Q, K, Q, (0, LD, D)),                     # k_out on q
    (Q, K, Q, (64, LD, D)),                    # k_out on q's second head
    (Q, K, (64, LD, D), (1 << 22, 64, D)),
    (Q, K, (72, LD, D), K),                    # q_out reaches into k
    (Q, K, FAR, (FAR[0] + 32, LD, D)),         # the outputs share half a head
    (Q, K, FAR, (FAR[0] + LD, LD, D)),         # and a token
    (Q, (64, LD, D), Q, (64, LD, D)),          # in place, k a head of q
    (Q, (0, LD, D), Q, (0, LD, D)),
])
def test_overlaps_are_refused(q, k, q_out, k_out):
    assert call(q, k, q_out, k_out) == ARG


def test_overlaps_with_the_read_only_inputs_are_refused():
    base = (1 << 20) + SIZE * FAR[0]
    for bad in (dict(pos=base), dict(pos=base + 8 * (3 * LD * SIZE // 8)), dict(table=base - 8 * D * 4 + 4), dict(weight=base)):
        assert call(Q, K, FAR, (1 << 22, 64, D), **bad) == ARG


def test_overlapping_output_rows_are_refused():
    for bad in ((FAR[0], 0, D), (FAR[0], LD, 32), (FAR[0], 96, D), (FAR[0], LD, 0)):
        assert call(Q, K, bad, (1 << 22, 64, D)) == SHAPE


@pytest.mark.gpu
def test_views_that_share_no_element():
    """q, k and v heads of one buffer in several orders, outputs in its free
    places: the bits of packed tensors."""
    import torch

    from minisgl_amd.kernel import rotary_qk

    dev = "cuda:0"
    gen = torch.Generator().manual_seed(1)
    T, G = 9, 3
    q, k = (torch.randn(T, G, D, generator=gen).bfloat16().to(dev) for _ in range(2))
    pos, table = torch.arange(T, device=dev), torch.randn(16, D, generator=gen).to(dev)
    want = rotary_qk(q.clone(), k.clone(), pos, table)

    def check(qv, kv, qo=None, ko=None):
        qv.copy_(q), kv.copy_(k)
        got = rotary_qk(qv, kv, pos, table, q_out=qo, k_out=ko)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

    def buffer(*shape):
        return torch.zeros(*shape, dtype=torch.bfloat16, device=dev)

    b = buffer(T, 3 * G, D)
    check(b[:, :G], b[:, G : 2 * G])                                    # q, k, v
    check(b[:, :G], b[:, G : 2 * G], None, b[:, 2 * G :])               # k to where v was
    b = buffer(T, G, 3, D)
    check(b[:, :, 0], b[:, :, 1])                                       # q, k, v of each group
    check(b[:, :, 0], b[:, :, 1], b[:, :, 2], None)
    b = buffer(2 * G, T, D)
    check(b[:G].transpose(0, 1), b[G:].transpose(0, 1))                 # heads outermost
    b = buffer(T, 2, G, D)
    check(q.clone(), k.clone(), b[:, 0], b[:, 1])                       # packed outputs
    b = buffer(2, T, G, D)
    check(q.clone(), k.clone(), b[0], b[1])
    b = buffer(2 * T, G, D)
    check(b[0::2], b[1::2])                                             # tokens in turn
    b = buffer(T + 40, G, 2, D)
    check(b[:T, :, 0], b[:T, :, 1], b[T : 2 * T, :, 0], b[2 * T : 3 * T, :, 1])


@pytest.mark.gpu
def test_overlapping_tensors_are_refused():
    import torch

    from minisgl_amd.kernel import MW8Error, rotary_qk

    dev = "cuda:0"
    b = torch.zeros(8, 4, D, dtype=torch.bfloat16, device=dev)
    pos, table = torch.arange(4, device=dev), torch.ones(8, D, device=dev)
    q, k = b[:4, :2], b[:4, 2:3]
    for kw in (dict(q_out=b.view(-1)[: 4 * 2 * D].view(4, 2, D)), dict(q_out=b[:4, 1:3]), dict(q_out=b[1:5, :2]),
               dict(k_out=b[:4, 1:2]), dict(k_out=b[1:5, 2:3])):
        with pytest.raises((MW8Error, ValueError), match="overlap"):
            rotary_qk(q, k, pos, table, **kw)
    with pytest.raises((MW8Error, ValueError), match="overlap"):
        rotary_qk(q, b[:4, 1:2], pos, table)
    assert not b.any()
