"""GPU parity of the rotary operators against the fp64 oracle.

Tolerance: one rounding to the element type, eps / 2 |y|, and fp32 arithmetic
on a c and b s: two products, one sum, and with a norm a sum of D squares, a
root, a quotient and two products, each off by at most 2^-24 of its value:
(D + 16) 2^-24 (|a c| + |b s|), with a subnormal step of the type on top."""

import numpy as np
import pytest
import torch

from helpers import announce
from minisgl_amd.kernel import rotary_cos_sin, rotary_qk
from oracle import rotary as orc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _table(P, R, scale=1.0, base=1e6):
    f = base ** (-np.arange(R // 2) * 2.0 / R)
    return torch.from_numpy(orc.table(f, P, scale)).float()


def _check(got, x, table, pos, inter, weight, eps, dtype):
    xv, tv, p = x.double().cpu().numpy(), table.double().numpy(), pos.cpu().numpy().astype(np.int64)
    w = None if weight is None else weight.double().cpu().numpy()
    want = orc.rotate(xv, tv, p, inter, w, eps)
    size = orc.rotate(np.abs(xv) if w is None else np.abs(orc.rotate(xv, np.concatenate(
        [np.ones((1, tv.shape[1] // 2)), np.zeros((1, tv.shape[1] // 2))], 1), np.zeros_like(p), inter, w, eps)),
        np.concatenate([np.abs(tv[:, : tv.shape[1] // 2]), -np.abs(tv[:, tv.shape[1] // 2 :])], 1), p, inter)
    # element b of a pair: |b c| + |a s|, with the sign of s turned back
    R = tv.shape[1]
    both = np.abs(size)
    for i in range(R // 2):
        ia, ib = (2 * i, 2 * i + 1) if inter else (i, R // 2 + i)
        c, s = np.abs(tv[p, i])[:, None], np.abs(tv[p, R // 2 + i])[:, None]
        base = xv if w is None else xv / np.sqrt((xv * xv).mean(-1, keepdims=True) + eps) * w
        both[..., ib] = np.abs(base[..., ib]) * c + np.abs(base[..., ia]) * s
    info = torch.finfo(dtype)
    tol = info.eps / 2 * np.abs(want) + (xv.shape[-1] + 16) * 2.0**-24 * both + info.smallest_normal * info.eps
    g = got.double().cpu().numpy()
    assert (np.abs(g - want) <= tol).all(), np.abs(g - want).max()


CASES = [
    # T, Hq, Hk, D, R
    (1, 1, 1, 2, 2), (1, 64, 8, 128, 128), (3, 5, 1, 80, 40), (7, 16, 2, 128, 64), (2, 4, 4, 64, 64), (33, 7, 1, 96, 96),
    (5, 3, 2, 256, 128), (4, 2, 1, 100, 50), (9, 1, 1, 18, 6), (300, 40, 8, 128, 128), (2, 2, 1, 576, 64), (17, 32, 4, 128, 32),
    (6, 130, 1, 64, 48), (3, 1, 3, 1000, 1000),
]


@pytest.mark.parametrize("T,hq,hk,D,R", CASES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dt", list(DTYPES))
def test_rotary(T, hq, hk, D, R, inter, norm, dt):
    announce(f"rotary T={T} Hq={hq} Hk={hk} D={D} R={R} inter={inter} norm={norm} {dt}")
    dtype = DTYPES[dt]
    gen = torch.Generator().manual_seed(T * 7 + D + R)
    qkv = torch.randn(T, (hq + 2 * hk) * D, generator=gen).to(dtype).to(DEV)
    before = qkv.clone()
    q, k = qkv[:, : hq * D].view(T, hq, D), qkv[:, hq * D : (hq + hk) * D].view(T, hk, D)
    table = _table(500, R, 1.1)
    pos = torch.randint(0, 500, (T,), generator=gen)
    pos[0] = 499
    if T % 2:
        pos = pos.int()
    w = [(torch.rand(D, generator=gen) + 0.5).to(dtype).to(DEV) if norm else None for _ in range(2)]
    args = (pos.to(DEV), table.to(DEV), inter, w[0], w[1], 1e-6)
    qo, ko = rotary_qk(q, k, *args, q_out=torch.empty(T, hq, D, dtype=dtype, device=DEV),
                       k_out=torch.empty(T, hk, D, dtype=dtype, device=DEV))
    assert torch.equal(qkv, before)
    _check(qo, q, table, pos, inter, w[0], 1e-6, dtype)
    _check(ko, k, table, pos, inter, w[1], 1e-6, dtype)
    q2, k2 = rotary_qk(q, k, *args)  # in place on the views
    assert q2 is q and torch.equal(q, qo) and torch.equal(k, ko)
    assert torch.equal(qkv[:, (hq + hk) * D :], before[:, (hq + hk) * D :])


@pytest.mark.parametrize("off,pad", [(0, 8), (8, 0), (1, 0), (4, 4), (0, 3)])
@pytest.mark.parametrize("inter", [False, True])
def test_rotary_strides_and_alignment(off, pad, inter):
    """Any token and head stride and any alignment: the bits of packed rows."""
    announce(f"rotary strides off={off} pad={pad}")
    T, H, D, R = 9, 5, 128, 96
    gen = torch.Generator().manual_seed(off + pad)
    x = torch.randn(T, H, D, generator=gen).bfloat16().to(DEV)
    kx = torch.randn(T, 1, D, generator=gen).bfloat16().to(DEV)
    table, pos = _table(64, R).to(DEV), torch.arange(T, device=DEV) * 3
    w = (torch.rand(D, generator=gen) + 0.5).bfloat16().to(DEV)
    want, kwant = x.clone(), kx.clone()
    rotary_qk(want, kwant, pos, table, inter, w, w)
    ld = H * (D + pad) + 16
    buf = torch.zeros(T * ld + 64, dtype=torch.bfloat16, device=DEV)
    v = buf[off:].as_strided((T, H, D), (ld, D + pad, 1))
    v.copy_(x)
    kv = kx.clone()
    rotary_qk(v, kv, pos, table, inter, w, w)
    assert torch.equal(v, want) and torch.equal(kv, kwant)
    # heads outermost ([H, T, D] seen as [T, H, D])
    ht = x.transpose(0, 1).contiguous().transpose(0, 1)
    rotary_qk(ht, kx.clone(), pos, table, inter, w, w)
    assert torch.equal(ht, want)


@pytest.mark.parametrize("D,R", [(128, 128), (128, 64), (18, 6)])
def test_rotary_padding_and_far_positions(D, R):
    announce(f"rotary padding and out of table D={D} R={R}")
    gen = torch.Generator().manual_seed(1)
    q, k = torch.randn(6, 4, D, generator=gen).bfloat16().to(DEV), torch.randn(6, 2, D, generator=gen).bfloat16().to(DEV)
    table = _table(32, R).to(DEV)
    ok = torch.tensor([0, 31, 5, 5, 7, 1], device=DEV)
    wq, wk = rotary_qk(q, k, ok, table, q_out=torch.empty_like(q), k_out=torch.empty_like(k))
    pos = torch.tensor([0, 31, -1, 32, 1 << 40, -(1 << 50)], device=DEV)
    qo, ko = torch.full_like(q, 9.0), torch.full_like(k, 9.0)
    rotary_qk(q, k, pos, table, q_out=qo, k_out=ko)
    for o, w, x in ((qo, wq, q), (ko, wk, k)):
        assert torch.equal(o[:2], w[:2])
        assert (o[2] == 9).all() and (o[5] == 9).all()
        assert torch.isnan(o[3, :, :R]).all() and torch.isnan(o[4, :, :R]).all()
        assert torch.equal(o[3:5, :, R:], x[3:5, :, R:])
    q[1, 2, 0], k[0, 0, R - 1] = float("nan"), float("inf")
    qo, ko = rotary_qk(q, k, ok, table, q_out=torch.empty_like(q), k_out=torch.empty_like(k))
    assert torch.isnan(qo[1, 2, [0, R // 2]]).all() and torch.equal(qo[0], wq[0]) and torch.equal(ko[1:], wk[1:])
    e = torch.empty(0, 4, D, dtype=torch.bfloat16, device=DEV)
    rotary_qk(e, e[:, :2], torch.empty(0, dtype=torch.int64, device=DEV), table)


def test_rotary_many_tokens():
    """More blocks than one axis of a grid holds, and rows past 2^31 bytes."""
    announce("rotary 70000 tokens x 130 heads")
    T, H, D = 70000, 130, 128
    q = torch.randn(T, 1, D, device=DEV).bfloat16().expand(T, H, D).contiguous()
    k = torch.zeros(T, 1, D, dtype=torch.bfloat16, device=DEV)
    table, pos = _table(4096, D).to(DEV), torch.arange(T, device=DEV) % 4096
    q1 = q[:, :1].clone()
    rotary_qk(q1, k.clone(), pos, table)
    rotary_qk(q, k, pos, table)
    assert torch.equal(q, q1.expand_as(q))


@pytest.mark.parametrize("P,half", [(1, 1), (1000, 64), (131072, 64), (257, 33), (4099, 3), (300, 500)])
def test_cos_sin_table(P, half):
    """fp64 angles: the table is off by fp32's rounding and the fp64 error of
    an angle up to 2^20 (2^-33), its functions' few ulps below that."""
    announce(f"rotary table P={P} pairs={half}")
    f = 1e6 ** (-np.arange(half) * 1.0 / half)
    t = rotary_cos_sin(torch.from_numpy(f).to(DEV), P, 1.25).double().cpu().numpy()
    want = orc.table(f, P, 1.25)
    assert t.shape == (P, 2 * half)
    assert (np.abs(t - want) <= 2.0**-24 * np.abs(want) + 1.25 * 2.0**-32).all()
    assert rotary_cos_sin(torch.from_numpy(f).to(DEV), 0).shape == (0, 2 * half)


def test_rotary_graph_and_stream():
    announce("rotary on a stream and in a graph")
    gen = torch.Generator().manual_seed(3)
    table = _table(512, 128).to(DEV)
    qs = [torch.randn(40, 8, 128, generator=gen).bfloat16().to(DEV) for _ in range(3)]
    ks = [torch.randn(40, 2, 128, generator=gen).bfloat16().to(DEV) for _ in range(3)]
    ps = [torch.randint(-1, 512, (40,), generator=gen).to(DEV) for _ in range(3)]
    want = [rotary_qk(q.clone(), k.clone(), p, table) for q, k, p in zip(qs, ks, ps)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = rotary_qk(qs[0].clone(), ks[0].clone(), ps[0], table)
    side.synchronize()
    assert torch.equal(got[0], want[0][0]) and torch.equal(got[1], want[0][1])
    q, k, p = qs[0].clone(), ks[0].clone(), ps[0].clone()
    qo, ko = torch.zeros_like(q), torch.zeros_like(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rotary_qk(q, k, p, table, q_out=qo, k_out=ko)
    for i in (1, 2, 0, 2):
        q.copy_(qs[i]), k.copy_(ks[i]), p.copy_(ps[i])
        qo.copy_(qs[i]), ko.copy_(ks[i])  # padding rows stay as they were
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(qo, want[i][0]) and torch.equal(ko, want[i][1])


def test_rotary_refusals():
    q, k = torch.zeros(4, 2, 64, device=DEV).bfloat16(), torch.zeros(4, 1, 64, device=DEV).bfloat16()
    pos, table = torch.arange(4, device=DEV), _table(8, 64).to(DEV)
    w = torch.ones(64, device=DEV).bfloat16()
    for call in (
        lambda: rotary_qk(q, k.float(), pos, table),
        lambda: rotary_qk(q, k[:3], pos, table),
        lambda: rotary_qk(q[0], k, pos, table),
        lambda: rotary_qk(q, k, pos.float(), table),
        lambda: rotary_qk(q, k, pos[:3], table),
        lambda: rotary_qk(q, k, pos.cpu(), table),
        lambda: rotary_qk(q, k, pos, table.double()),
        lambda: rotary_qk(q, k, pos, table[:, :63].contiguous()),
        lambda: rotary_qk(q, k, pos, _table(8, 128).to(DEV)),
        lambda: rotary_qk(q, k, pos, table, q_weight=w.float()),
        lambda: rotary_qk(q, k, pos, table, k_weight=w[:32]),
        lambda: rotary_qk(q, k, pos, table, q_out=q[:, :1]),
        lambda: rotary_qk(q, q, pos, table),
        lambda: rotary_qk(q.transpose(1, 2), k, pos, table),
        lambda: rotary_qk(q[:, :1].expand(4, 2, 64), k, pos, table),
        lambda: rotary_cos_sin(torch.ones(4, device=DEV), 8),
        lambda: rotary_cos_sin(torch.ones(4, dtype=torch.float64), 8),
        lambda: rotary_cos_sin(torch.ones(4, dtype=torch.float64, device=DEV), -1),
    ):
        with pytest.raises(ValueError):
            call()


def test_rotary_refuses_crossed_outputs_and_sizes_past_the_entry():
    """An output on the other input; a head, head count or frequency list
    that a 32-bit argument cannot hold (views of a little memory)."""
    q, k = (torch.zeros(4, h, 64, dtype=torch.bfloat16, device=DEV) for h in (2, 2))
    pos, table = torch.arange(4, device=DEV), torch.ones(8, 64, device=DEV)
    out = torch.zeros_like(q)
    one = torch.zeros(1, dtype=torch.bfloat16, device=DEV)
    for call in (
        lambda: rotary_qk(q, k, pos, table, q_out=k, k_out=out),
        lambda: rotary_qk(q, k, pos, table, q_out=out, k_out=q),
        lambda: rotary_qk(one.expand(1, 1, 2**32 + 64), one.expand(1, 1, 2**32 + 64), pos[:1], table),
        lambda: rotary_qk(one.expand(1, 2**32 + 1, 64), one.expand(1, 1, 64), pos[:1], table),
        lambda: rotary_cos_sin(torch.ones(4097, dtype=torch.float64, device=DEV), 8),
    ):
        with pytest.raises(ValueError):
            call()
    assert not out.any()


@pytest.mark.parametrize("D,R", [(128, 64), (100, 50)])
def test_rotary_one_sided(D, R):
    """No key heads, no query heads, no heads; a norm of one of the two."""
    announce(f"rotary one-sided D={D} R={R}")
    gen = torch.Generator().manual_seed(D)
    q, k = (torch.randn(5, h, D, generator=gen).bfloat16().to(DEV) for h in (3, 2))
    table, pos = _table(16, R).to(DEV), torch.arange(5, device=DEV)
    w = (torch.rand(D, generator=gen) + 0.5).bfloat16().to(DEV)
    plain = rotary_qk(q.clone(), k.clone(), pos, table)
    normed = rotary_qk(q.clone(), k.clone(), pos, table, q_weight=w, k_weight=w)
    for kw, pick in (({"q_weight": w}, (normed[0], plain[1])), ({"k_weight": w}, (plain[0], normed[1]))):
        got = rotary_qk(q.clone(), k.clone(), pos, table, **kw)
        assert torch.equal(got[0], pick[0]) and torch.equal(got[1], pick[1])
    got = rotary_qk(q.clone(), k[:, :0], pos, table)
    assert torch.equal(got[0], plain[0]) and got[1].shape == (5, 0, D)
    assert torch.equal(rotary_qk(q[:, :0], k.clone(), pos, table)[1], plain[1])
    rotary_qk(q[:, :0], k[:, :0], pos, table)


def test_rotary_head_major_views():
    """Tensors stored [heads, T, D], read as [T, heads, D], in place and into
    another order."""
    announce("rotary head-major")
    gen = torch.Generator().manual_seed(9)
    q, k = (torch.randn(6, h, 64, generator=gen).bfloat16().to(DEV) for h in (4, 2))
    table, pos = _table(16, 64).to(DEV), torch.arange(6, device=DEV)
    want = rotary_qk(q.clone(), k.clone(), pos, table)
    qh, kh = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k))
    out = rotary_qk(qh, kh, pos, table, q_out=torch.empty_like(q, memory_format=torch.contiguous_format),
                    k_out=torch.empty_like(k, memory_format=torch.contiguous_format))
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    rotary_qk(qh, kh, pos, table)
    assert torch.equal(qh, want[0]) and torch.equal(kh, want[1])
