"""The MXFP4 and rotary layers as a decoder layer runs them: norm +
quantizer -> qkv -> per-head norm + rotation -> o_proj -> norm + residual +
quantizer -> gated MLP.  Each stage is compared with the fp64 oracle on the
stage's own inputs; the whole is captured, replayed with other batches
(padded ones among them) and compared with the eager run bit for bit."""

import numpy as np
import pytest
import torch

from helpers import announce, f32
from minisgl_amd.kernel import dequant_mxfp4, rmsnorm_quant
from minisgl_amd.layers import GatedMLPMXFP4, LinearMXFP4, RMSNorm, RMSNormQuantMXFP4, RotaryEmbedding
from oracle import mxfp4 as orc
from oracle import rotary as rorc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-6


class Layer:
    """The parts of a decoder layer around attention (q stands in for its output)."""

    def __init__(self, hidden, inter, heads, kv, dim, seed, rotary_dim=None, interleaved=False):
        gen = torch.Generator().manual_seed(seed)
        self.heads, self.kv, self.dim = heads, kv, dim

        def weight(n, k):
            return (torch.randn(n, k, generator=gen) / k**0.5).bfloat16().to(DEV)

        def norm(cls, size):
            layer = cls(size, EPS)
            layer.load_state_dict({"weight": (torch.rand(size, generator=gen) + 0.5).bfloat16().to(DEV)})
            return layer

        self.norm1, self.norm2 = norm(RMSNormQuantMXFP4, hidden), norm(RMSNormQuantMXFP4, hidden)
        self.q_norm, self.k_norm = norm(RMSNorm, dim), norm(RMSNorm, dim)
        self.qkv = LinearMXFP4(hidden, [heads * dim, kv * dim, kv * dim], has_bias=True)
        n = (heads + 2 * kv) * dim
        self.qkv.load_float_weight(weight(n, hidden), torch.randn(n, generator=gen).to(DEV))
        self.o = LinearMXFP4(heads * dim, hidden)
        self.o.load_float_weight(weight(hidden, heads * dim))
        self.mlp = GatedMLPMXFP4(hidden, inter)
        self.mlp.gate_up_proj.load_float_weight(weight(2 * inter, hidden))
        self.mlp.down_proj.load_float_weight(weight(hidden, inter))
        self.rope = RotaryEmbedding(dim, rotary_dim or dim, 4096, 1e6, {"rope_type": "yarn", "factor": 4.0,
                                    "original_max_position_embeddings": 1024}, interleaved)

    def run(self, x, residual, positions, keep=None):
        codes, scale, residual = self.norm1.forward(x, residual)
        qkv = self.qkv.forward_quantized(codes, scale)
        if keep is not None:
            keep.update(c1=(codes, scale), r1=residual.clone(), qkv=qkv.clone())
        q, k, v = qkv.split([self.heads * self.dim, self.kv * self.dim, self.kv * self.dim], 1)
        self.rope.forward(positions, q, k, self.q_norm, self.k_norm)
        attn = self.o.forward(q)
        codes, scale, residual = self.norm2.forward(attn, residual)
        y = self.mlp.forward_quantized(codes, scale)
        if keep is not None:
            keep.update(rot=qkv.clone(), attn=attn, r2=residual, c2=(codes, scale))
        return y, residual, qkv


def _values(pair, K):
    from minisgl_amd.kernel import mxfp4_row_scales

    byte = mxfp4_row_scales(pair[1], K).cpu().numpy()
    return orc.values(orc.unpack(pair[0].cpu().numpy()), byte)


def _close(got, want, size, K):
    tol = 2.0**-8 * np.abs(want) + (K + 1) * 2.0**-23 * size
    assert (np.abs(f32(got).astype(np.float64) - want) <= tol).all()


@pytest.mark.parametrize("M,shape", [
    (1, dict(hidden=1024, inter=768, heads=8, kv=2, dim=128)),
    (7, dict(hidden=1000, inter=500, heads=5, kv=1, dim=80, rotary_dim=40, interleaved=True)),
    (65, dict(hidden=512, inter=640, heads=4, kv=4, dim=64)),
    (300, dict(hidden=1024, inter=1536, heads=8, kv=1, dim=128, rotary_dim=64)),
    (1100, dict(hidden=512, inter=2048, heads=4, kv=2, dim=128)),
])
def test_decoder_layer_stages(M, shape):
    announce(f"mxfp4 decoder layer M={M} {shape}")
    layer = Layer(seed=M, **shape)
    gen = torch.Generator().manual_seed(M)
    hidden, inter, dim = shape["hidden"], shape["inter"], shape["dim"]
    x, res = (torch.randn(M, hidden, generator=gen).bfloat16().to(DEV) for _ in range(2))
    pos = torch.randint(0, 4096, (M,), generator=gen)
    want_r, xs = res.clone(), x.clone()
    want_y = rmsnorm_quant(xs, layer.norm1.weight, EPS, residual=want_r, quantize=False)
    keep = {}
    y, r2, _ = layer.run(x, res, pos.to(DEV), keep)
    # norm1: the framework's own norm, then the oracle's codes of its output
    assert torch.equal(keep["r1"], want_r)
    code, byte = orc.quantize(f32(want_y).astype(np.float64))
    np.testing.assert_array_equal(keep["c1"][0].cpu().numpy(), orc.pack(code))
    # qkv
    w = _values((layer.qkv.weight, layer.qkv.weight_scale), hidden)
    want, size = orc.product(orc.values(code, byte), w, f32(layer.qkv.bias).astype(np.float64))
    _close(keep["qkv"], want, size, hidden)
    # rotation of the qkv product as it was
    table = layer.rope.prepare(torch.device(DEV)).double().cpu().numpy()
    n, kn = layer.heads * dim, layer.kv * dim
    before, after = (f32(keep[k]).astype(np.float64) for k in ("qkv", "rot"))
    for lo, hi, norm in ((0, n, layer.q_norm), (n, n + kn, layer.k_norm)):
        want = rorc.rotate(before[:, lo:hi].reshape(M, -1, dim), table, pos.numpy(), layer.rope.interleaved,
                           f32(norm.weight).astype(np.float64), EPS).reshape(M, -1)
        big = np.abs(want).max()
        assert (np.abs(after[:, lo:hi] - want) <= 2.0**-8 * np.abs(want) + (dim + 16) * 2.0**-24 * 4 * big).all()
    np.testing.assert_array_equal(after[:, n + kn:], before[:, n + kn:])
    # o_proj of the rotated q
    w = _values((layer.o.weight, layer.o.weight_scale), n)
    want, size = orc.product(orc.values(*orc.quantize(after[:, :n])), w)
    _close(keep["attn"], want, size, n)
    # the MLP on the second norm's codes
    v2 = _values(keep["c2"], hidden)
    w1 = _values((layer.mlp.gate_up_proj.weight, layer.mlp.gate_up_proj.weight_scale), hidden)
    gu = orc.round_bf16(orc.product(v2, w1)[0])
    h = orc.round_bf16(orc.activation(gu[:, :inter], "silu") * gu[:, inter:])
    w2 = _values((layer.mlp.down_proj.weight, layer.mlp.down_proj.weight_scale), inter)
    want = orc.product(orc.values(*orc.quantize(h)), w2)[0]
    # fewer than 1 in 1000 codes of h may change by a third (see the gated MLP's test)
    assert np.linalg.norm(f32(y) - want) <= 0.02 * np.linalg.norm(want)
    # the same codes as values: the MLP that quantizes its input itself (these values quantize to themselves)
    assert torch.equal(layer.mlp.forward(dequant_mxfp4(*keep["c2"], hidden)), y)


@pytest.mark.parametrize("M", [1, 8, 64, 256])
def test_decoder_layer_in_a_graph(M):
    """Captured once, replayed with full and padded batches between eager runs:
    the bits of the eager run; a padded row leaves the others alone."""
    announce(f"mxfp4 decoder layer in a graph M={M}")
    layer = Layer(hidden=1024, inter=768, heads=8, kv=2, dim=128, seed=1)
    gen = torch.Generator().manual_seed(M)
    sets = []
    for i in range(3):
        pos = torch.randint(0, 4096, (M,), generator=gen)
        if i == 1:
            pos[M // 2:] = -1
        sets.append([torch.randn(M, 1024, generator=gen).bfloat16().to(DEV), torch.randn(M, 1024, generator=gen).bfloat16().to(DEV),
                     pos.to(DEV)])
    want = [layer.run(x.clone(), r.clone(), p) for x, r, p in sets]
    x, r, p = (t.clone() for t in sets[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.run(x, r, p)
    for i in (1, 2, 0, 1):
        for dst, src in zip((x, r, p), sets[i]):
            dst.copy_(src)
        graph.replay()
        eager = layer.run(*(t.clone() for t in sets[(i + 1) % 3]))
        torch.cuda.synchronize()
        for g, e, w, o in zip(out, eager, want[(i + 1) % 3], want[i]):
            assert torch.equal(e, w) and torch.equal(g, o)


def test_rotary_layer_refuses_its_first_use_in_a_capture():
    rope = RotaryEmbedding(64, 64, 16, 1e4)
    q, k, p = torch.zeros(2, 128, device=DEV).bfloat16(), torch.zeros(2, 64, device=DEV).bfloat16(), torch.arange(2, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="prepare"):
        with torch.cuda.graph(graph):
            rope.forward(p, q, k)
    torch.cuda.synchronize()
    a = rope.prepare(torch.device(DEV))
    assert rope.prepare(torch.device("cuda")) is a and a.shape == (16, 64)
    rope.forward(p, q, k)
    with pytest.raises(ValueError, match="eps"):
        rope.forward(p, q, k, RMSNorm(64, 1e-5), RMSNorm(64, 1e-6))
    with pytest.raises(ValueError, match="heads"):
        rope.forward(p, q[:, :100], k)
    rope.forward(p[:0], q[:0], k[:0])


def test_norm_layer_with_strided_residual():
    """A residual that is a view of a wider buffer is updated through it."""
    norm = RMSNormQuantMXFP4(256, EPS)
    norm.load_state_dict({"weight": torch.ones(256, dtype=torch.bfloat16, device=DEV)})
    x = torch.randn(5, 256, device=DEV).bfloat16()
    wide = torch.randn(5, 300, device=DEV).bfloat16()
    plain = wide[:, :256].contiguous()
    c1, s1, r1 = norm.forward(x, plain)
    c2, s2, r2 = norm.forward(x, wide[:, :256])
    assert torch.equal(c1, c2) and torch.equal(s1, s2) and torch.equal(r1, wide[:, :256]) and r2.data_ptr() == wide.data_ptr()
