"""The MXFP4 and rotary operators of a decoder layer, as timed cases.

Each case is one call (or the few calls) that a model runner makes: the
microscaled 4-bit quantizer and its inverse, a linear from bf16 rows, the
product of operands that are quantized already, the gated MLP, the input
half of an attention block (norm, quantization, qkv product, per-head norm
and rotation), the rotation by itself and the rotary table.  ``listed``
names the fixed cases, ``draw`` gives more of the same ranges.

With ``own`` false ``run`` computes the plain forms in elementary torch
operations, in 32 bits and rounded where the operators' definitions round
(the quantizers' codes, the bf16 tensors between two operators of a chain).

MXFP4: blocks of 32 elements along K share a power-of-two scale 2^e, e =
floor(log2(amax)) - 2 held as a byte e + 127 in [0, 254]; an element is an
e2m1 value (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), rounded to
nearest even, saturating.  Codes are packed two per byte, the even element
in the low half.  Scales travel in the layout [ceil(K / 512), rows, 16]: of
the 16 blocks of 512 elements, block 8 t + 2 g + s is byte 4 g + 2 t + s.

Weights are N(0, 1/K), quantized as above; activations are N(0, 1) in bf16
with 0.1% of the entries 20 times larger.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
HEAD = 128
EPS = 1e-6

# hidden, intermediate, query heads, key/value heads
QWEN3_14B = dict(hidden=5120, inter=17408, heads=40, kv=8)
QWEN3_32B = dict(hidden=5120, inter=25600, heads=64, kv=8)
QWEN3_32B_TP4 = dict(hidden=5120, inter=6400, heads=16, kv=2)  # one of four ranks' share
QWEN3_30B_A3B = dict(hidden=2048, inter=768, heads=32, kv=4)
MODELS = (QWEN3_14B, QWEN3_32B, QWEN3_32B_TP4, QWEN3_30B_A3B)

LARGEST = 8192 * 34816 * 5120  # multiplications of the largest product


def _kernels():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-sglang-fork_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from minisgl_amd import kernel

    return kernel


def listed():
    return [
        # a ragged batch of short rows, the last block of each partly filled
        dict(name="quant_m333_k1000", kind="quant", m=333, k=1000),
        # the largest prefill's MLP activation
        dict(name="quant_8192x17408", kind="quant", m=8192, k=17408),
        # one token through qkv: the latency of single-stream decode
        dict(name="linear_m1_qkv", kind="linear", m=1, k=5120, n=7168, bias=False),
        # a decode batch through the deep projection
        dict(name="linear_m64_down", kind="linear", m=64, k=17408, n=5120, bias=False),
        # the ragged tail of a chunked prefill through qkv with a bias
        dict(name="linear_m333_bias", kind="linear", m=333, k=5120, n=7168, bias=True),
        # the largest prefill batch through gate_up, operands quantized by the norm before it
        dict(name="product_m8192", kind="product", m=8192, k=5120, n=34816),
        # a decode batch through the gated MLP
        dict(name="mlp_m16", kind="mlp", m=16, act="silu", hidden=5120, inter=17408),
        # 32 decode tokens beside a 2048-token prefill chunk through the gated MLP
        dict(name="mlp_m2080", kind="mlp", m=2080, act="silu", hidden=5120, inter=25600),
        # one token from the residual stream to rotated q and k
        dict(name="attn_in_m1", kind="attn_in", m=1, hidden=5120, heads=64, kv=8),
        # a prefill chunk beside decode tokens, one of four ranks' share
        dict(name="attn_in_m2080", kind="attn_in", m=2080, hidden=5120, heads=16, kv=2),
        # a long prefill's q and k by themselves: interleaved pairs, half of each head, fp16
        dict(name="rotary_t8000_part", kind="rotary", m=8000, heads=32, kv=8, dim=128, part=64, interleaved=True, norm=False,
             dtype="float16"),
        # the table of a context of 131072 tokens
        dict(name="table_131072", kind="table", positions=131072, part=128),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choices(["quant", "linear", "product", "mlp", "attn_in", "rotary", "table"], [2, 5, 2, 4, 3, 3, 1])[0]
    m = _log_int(rng, 1, 8192)
    if kind == "quant":
        return dict(kind=kind, m=m, k=_log_int(rng, 8, 17408))
    if kind in ("linear", "product"):
        c = rng.choice(MODELS)
        h, i, qkv = c["hidden"], c["inter"], (c["heads"] + 2 * c["kv"]) * HEAD
        if rng.random() < 0.6:
            k, n = rng.choice([(h, qkv), (c["heads"] * HEAD, h), (h, 2 * i), (i, h)])
        else:
            k, n = 32 * _log_int(rng, 2, 512), _log_int(rng, 64, 32768)
        while m * k * n > LARGEST:
            m //= 2
        if kind == "product":
            return dict(kind=kind, m=m, k=k, n=n)
        return dict(kind=kind, m=m, k=k, n=n, bias=rng.random() < 0.3)
    if kind == "mlp":
        c = rng.choice(MODELS)
        m = min(m, LARGEST // (3 * c["hidden"] * c["inter"]))
        return dict(kind=kind, m=m, act=rng.choice(["silu", "silu", "gelu"]), hidden=c["hidden"], inter=c["inter"])
    if kind == "attn_in":
        c = rng.choice(MODELS)
        return dict(kind=kind, m=m, hidden=c["hidden"], heads=c["heads"], kv=c["kv"])
    if kind == "table":
        return dict(kind=kind, positions=_log_int(rng, 1000, 131072), part=rng.choice([32, 64, 96, 128]))
    dim = rng.choice([64, 80, 128, 256])
    part = rng.choice([dim, dim, dim // 2])
    heads, kv = rng.choice([(40, 8), (64, 8), (16, 2), (32, 4), (7, 1)])
    return dict(kind=kind, m=m, heads=heads, kv=kv, dim=dim, part=part, interleaved=rng.random() < 0.5, norm=rng.random() < 0.4,
                dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]))


# ------------------------------------------------------------------ inputs
def _acts(m, k, gen):
    x = torch.randn((m, k), generator=gen, device=DEV, dtype=torch.bfloat16)
    x[torch.rand((m, k), generator=gen, device=DEV) < 1e-3] *= 20
    return x


def _codes(v):
    """fp32 [m, k], k a multiple of 32 -> (packed codes [m, k / 2], scale bytes [m, k / 32])."""
    m, k = v.shape
    blocks = v.view(m, k // 32, 32)
    amax = blocks.abs().amax(2)
    scale = ((amax.view(torch.int32) >> 23) - 2).clamp(min=0)
    a = (blocks * torch.exp2((127 - scale).double()).float()[:, :, None]).reshape(m, k)
    mag = a.abs()
    code = (a.signbit()).to(torch.uint8) * 8
    code += mag > 0.25
    code += mag >= 0.75
    code += mag > 1.25
    code += mag >= 1.75
    code += mag > 2.5
    code += mag >= 3.5
    code += mag > 5
    return code[:, 0::2] | (code[:, 1::2] << 4), scale.to(torch.uint8)


def _tiles(scale):
    """Scale bytes [m, k / 32] -> the layout that they travel in."""
    m, kb = scale.shape
    t = -(-kb // 16)
    s = torch.zeros((m, t * 16), dtype=torch.uint8, device=scale.device)
    s[:, :kb] = scale
    return s.view(m, t, 2, 4, 2).permute(1, 0, 3, 2, 4).contiguous().view(t, m, 16)


def _weight(n, k, gen):
    """A weight [n, k] as a program holds it: packed codes, scale bytes, and these in the layout of the product."""
    kp = -(-k // 32) * 32
    codes = torch.empty((n, kp // 2), dtype=torch.uint8, device=DEV)
    scale = torch.empty((n, kp // 32), dtype=torch.uint8, device=DEV)
    for r in range(0, n, 8192):
        e = min(n, r + 8192)
        v = torch.zeros((e - r, kp), device=DEV)
        v[:, :k] = torch.randn((e - r, k), generator=gen, device=DEV) / math.sqrt(k)
        codes[r:e], scale[r:e] = _codes(v)
    return codes, scale, _tiles(scale)


def _frequencies(part, base=1e6, factor=4.0, original=32768, fast=32.0, slow=1.0):
    """Inverse frequencies of a context stretched `factor` times (YaRN): those that turn often stay, those that turn
    less than once over the original context are divided, a ramp between."""
    i = torch.arange(part // 2, dtype=torch.float64)
    f = base ** (-2 * i / part)

    def at(turns):
        return part * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), part - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return (f / factor * ramp + f * (1 - ramp)).to(DEV)


ATTENTION = 0.1 * math.log(4.0) + 1.0  # what a context stretched 4 times scales cos and sin by


def _table(freq, positions, scale):
    t = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * freq
    return (torch.cat([t.cos(), t.sin()], 1) * scale).float()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)
    st = dict(case=case)
    kind = case["kind"]
    if kind == "quant":
        st["x"] = _acts(case["m"], case["k"], gen)
    elif kind == "linear":
        st["x"] = _acts(case["m"], case["k"], gen)
        st["w"] = _weight(case["n"], case["k"], gen)
        st["bias"] = torch.randn(case["n"], generator=gen, device=DEV, dtype=torch.bfloat16) if case["bias"] else None
    elif kind == "product":
        codes, scale = _codes(_acts(case["m"], case["k"], gen).float())
        st["a"] = (codes, scale, _tiles(scale))
        st["w"] = _weight(case["n"], case["k"], gen)
    elif kind == "mlp":
        st["x"] = _acts(case["m"], case["hidden"], gen)
        st["w1"] = _weight(2 * case["inter"], case["hidden"], gen)
        st["w2"] = _weight(case["hidden"], case["inter"], gen)
    elif kind == "attn_in":
        n = (case["heads"] + 2 * case["kv"]) * HEAD
        st["x"] = _acts(case["m"], case["hidden"], gen)
        st["w"] = _weight(n, case["hidden"], gen)
        st["norm"] = (torch.rand(case["hidden"], generator=gen, device=DEV) * 1.5 + 0.25).bfloat16()
        st["q_norm"] = (torch.rand(HEAD, generator=gen, device=DEV) * 1.5 + 0.25).bfloat16()
        st["k_norm"] = (torch.rand(HEAD, generator=gen, device=DEV) * 1.5 + 0.25).bfloat16()
        st["table"] = _table(_frequencies(HEAD), 40960, ATTENTION)
        st["pos"] = torch.randint(0, 40960, (case["m"],), generator=gen, device=DEV)
    elif kind == "rotary":
        dtype = getattr(torch, case["dtype"])
        heads, kv, dim = case["heads"], case["kv"], case["dim"]
        qkv = torch.randn((case["m"], (heads + 2 * kv) * dim), generator=gen, device=DEV).to(dtype)
        st["q"] = qkv[:, : heads * dim].view(-1, heads, dim)
        st["k"] = qkv[:, heads * dim : (heads + kv) * dim].view(-1, kv, dim)
        st["q_out"] = torch.empty((case["m"], heads, dim), dtype=dtype, device=DEV)
        st["k_out"] = torch.empty((case["m"], kv, dim), dtype=dtype, device=DEV)
        st["q_norm"] = (torch.rand(dim, generator=gen, device=DEV) * 1.5 + 0.25).to(dtype) if case["norm"] else None
        st["k_norm"] = (torch.rand(dim, generator=gen, device=DEV) * 1.5 + 0.25).to(dtype) if case["norm"] else None
        st["table"] = _table(_frequencies(case["part"]), 40960, ATTENTION)
        st["pos"] = torch.randint(0, 40960, (case["m"],), generator=gen, device=DEV)
    else:
        # the seed picks the stretch of the context
        st["freq"] = _frequencies(case["part"], factor=2.0 + torch.rand(1, generator=gen, device=DEV).item() * 6.0)
    return st


# ------------------------------------------------------------- plain forms
def _values(codes, scale):
    """Packed codes and scale bytes -> fp32 values."""
    level = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = torch.empty((codes.shape[0], codes.shape[1] * 2), device=codes.device)
    v[:, 0::2] = level[(codes & 15).int()]
    v[:, 1::2] = level[(codes >> 4).int()]
    return v * torch.exp2(scale.double() - 127).float().repeat_interleave(32, 1)


def _padded(x):
    """fp32 rows with zeros up to a whole block."""
    return torch.nn.functional.pad(x.float(), (0, -x.shape[1] % 32))


def _product(a, w, bias=None):
    y = a @ _values(w[0], w[1]).T
    return (y if bias is None else y + bias.float()).bfloat16()


def _quantized(x):
    return _values(*_codes(_padded(x)))


def _rms(x, weight, eps):
    """x / rms(x) * weight over the last axis, in fp32 (the sum of squares in 64 bits)."""
    x = x.float()
    r = 1 / torch.sqrt(x.double().square().mean(-1, keepdim=True).float() + eps)
    return x * r * weight.float()


def _activation(g, act):
    return g * torch.sigmoid(g) if act == "silu" else 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))


def _rotated(x, table, pos, part, interleaved, weight=None):
    """x [t, heads, dim] with the first `part` elements of each head turned by its position's angles."""
    v = x.float() if weight is None else _rms(x, weight, EPS)
    cos, sin = table[pos].view(-1, 1, 2, part // 2).unbind(2)
    if interleaved:
        a, b = v[..., 0:part:2], v[..., 1:part:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = v[..., : part // 2], v[..., part // 2 : part]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, v[..., part:]], -1).to(x.dtype)


def _run_plain(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "quant":
        return _quantized(st["x"])[:, : case["k"]].bfloat16()
    if kind == "linear":
        return _product(_quantized(st["x"]), st["w"], st["bias"])
    if kind == "product":
        return _product(_values(st["a"][0], st["a"][1]), st["w"])
    if kind == "mlp":
        gu = _product(_quantized(st["x"]), st["w1"]).float()
        h = (_activation(gu[:, : case["inter"]], case["act"]) * gu[:, case["inter"] :]).bfloat16()
        return _product(_quantized(h), st["w2"])
    if kind == "attn_in":
        h = _rms(st["x"], st["norm"], EPS).bfloat16()
        qkv = _product(_quantized(h), st["w"])
        q, k, v = qkv.split([case["heads"] * HEAD, case["kv"] * HEAD, case["kv"] * HEAD], 1)
        q = _rotated(q.view(-1, case["heads"], HEAD), st["table"], st["pos"], HEAD, False, st["q_norm"])
        k = _rotated(k.view(-1, case["kv"], HEAD), st["table"], st["pos"], HEAD, False, st["k_norm"])
        return q, k, v
    if kind == "rotary":
        return tuple(_rotated(st[n], st["table"], st["pos"], case["part"], case["interleaved"], st[n + "_norm"]) for n in "qk")
    return _table(st["freq"], case["positions"], ATTENTION)


# ------------------------------------------------------ the framework's own
def _run_own(st):
    kn = _kernels()
    case = st["case"]
    kind = case["kind"]
    if kind == "quant":
        codes, scale = kn.quant_mxfp4(st["x"])
        return kn.dequant_mxfp4(codes, scale, case["k"])
    if kind == "linear":
        return kn.linear_mxfp4(st["x"], st["w"][0], st["w"][2], st["bias"])
    if kind == "product":
        return kn.gemm_mxfp4(st["a"][0], st["a"][2], st["w"][0], st["w"][2])
    if kind == "mlp":
        return kn.gated_mlp_mxfp4(st["x"], st["w1"][0], st["w1"][2], st["w2"][0], st["w2"][2], case["act"])
    if kind == "attn_in":
        codes, scale = kn.rmsnorm_quant_mxfp4(st["x"], st["norm"], EPS)
        qkv = kn.gemm_mxfp4(codes, scale, st["w"][0], st["w"][2])
        q, k, v = qkv.split([case["heads"] * HEAD, case["kv"] * HEAD, case["kv"] * HEAD], 1)
        q, k = q.view(-1, case["heads"], HEAD), k.view(-1, case["kv"], HEAD)
        kn.rotary_qk(q, k, st["pos"], st["table"], q_weight=st["q_norm"], k_weight=st["k_norm"], eps=EPS)
        return q, k, v
    if kind == "rotary":
        return kn.rotary_qk(st["q"], st["k"], st["pos"], st["table"], interleaved=case["interleaved"], q_weight=st["q_norm"],
                            k_weight=st["k_norm"], eps=EPS, q_out=st["q_out"], k_out=st["k_out"])
    return kn.rotary_cos_sin(st["freq"], case["positions"], ATTENTION)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# -------------------------------------------------------------------- work
def _operand(rows, k):
    """Bytes of a quantized matrix."""
    return rows * -(-k // 32) * 17


def work(case):
    kind = case["kind"]
    if kind == "quant":
        # the rows read, their values written
        return dict(bytes=4 * case["m"] * case["k"], flops=2 * case["m"] * case["k"])
    if kind in ("linear", "product"):
        m, k, n = case["m"], case["k"], case["n"]
        read = 2 * m * k if kind == "linear" else _operand(m, k)
        return dict(bytes=read + _operand(n, k) + 2 * m * n + (2 * n if case.get("bias") else 0), flops=2 * m * n * k)
    if kind == "mlp":
        m, h, i = case["m"], case["hidden"], case["inter"]
        return dict(bytes=4 * m * h + _operand(2 * i, h) + _operand(h, i), flops=6 * m * h * i)
    if kind == "attn_in":
        m, h, n = case["m"], case["hidden"], (case["heads"] + 2 * case["kv"]) * HEAD
        return dict(bytes=2 * m * h + _operand(n, h) + 2 * m * n + 4 * m * HEAD, flops=2 * m * h * n)
    if kind == "rotary":
        size = {"float32": 4}.get(case["dtype"], 2)
        rows = case["m"] * (case["heads"] + case["kv"])
        return dict(bytes=2 * rows * case["dim"] * size + case["m"] * (4 * case["part"] + 8), flops=3 * rows * case["part"])
    return dict(bytes=4 * case["positions"] * case["part"], flops=40 * case["positions"] * case["part"])


# ---------------------------------------------------------------- 64 bits
def _exact_quantized(x):
    """The quantizer's values in 64 bits, from its definition."""
    m, k = x.shape
    v = torch.zeros((m, -(-k // 32), 32), dtype=torch.float64, device=x.device)
    v.view(m, -1)[:, :k] = x.double()
    amax = v.abs().amax(2, keepdim=True)
    e = (torch.frexp(amax).exponent - 3).clamp(-127, 127)  # floor(log2(amax)) - 2
    e = torch.where(amax == 0, torch.full_like(e, -127), e).double()
    a = v * torch.exp2(-e)
    step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
    return ((torch.round(a / step) * step).clamp(-6, 6) * torch.exp2(e)).view(m, -1)


def _exact_operand(packed):
    codes, scale = packed[0].long(), packed[1].double()
    both = torch.stack([codes % 16, codes // 16], 2).flatten(1)
    c = both % 8
    # e2m1: exponent c / 2, mantissa c % 2; exponent 0 is 0 or 0.5
    mag = torch.where(c < 2, 0.5 * c.double(), (1 + 0.5 * (c % 2).double()) * torch.exp2((c // 2 - 1).double()))
    s = torch.repeat_interleave(torch.exp2(scale - 127), 32, dim=1)
    return torch.where(both >= 8, -mag, mag) * s


def _exact_product(a, packed):
    out = []
    for r in range(0, packed[0].shape[0], 8192):
        out.append(a @ _exact_operand([t[r : r + 8192] for t in packed[:2]]).T)
    return torch.cat(out, 1)


def _exact_rms(x, weight):
    v = x.double()
    return v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS) * weight.double()


def _exact_rotated(v, table, pos, part, interleaved):
    half = part // 2
    z = torch.complex(table[pos][:, None, :half].double(), table[pos][:, None, half:].double())
    if interleaved:
        turned = torch.view_as_real(torch.view_as_complex(v[..., :part].unflatten(-1, (half, 2)).contiguous()) * z).flatten(-2)
    else:
        w = torch.complex(v[..., :half].contiguous(), v[..., half:part].contiguous()) * z
        turned = torch.cat([w.real, w.imag], -1)
    return torch.cat([turned, v[..., part:]], -1)


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "quant":
        return _exact_quantized(st["x"])[:, : case["k"]]
    if kind == "linear":
        y = _exact_product(_exact_quantized(st["x"]), st["w"])
        return y if st["bias"] is None else y + st["bias"].double()
    if kind == "product":
        return _exact_product(_exact_operand(st["a"]), st["w"])
    if kind == "mlp":
        gu = _exact_product(_exact_quantized(st["x"]), st["w1"]).bfloat16().double()
        g, u = gu.chunk(2, 1)
        h = g / (1 + torch.exp(-g)) if case["act"] == "silu" else g * 0.5 * torch.erfc(-g / math.sqrt(2))
        return _exact_product(_exact_quantized((h * u).bfloat16()), st["w2"])
    if kind == "attn_in":
        qkv = _exact_product(_exact_quantized(_exact_rms(st["x"], st["norm"]).bfloat16()), st["w"]).bfloat16()
        heads, kv = case["heads"], case["kv"]
        q, k, v = qkv.split([heads * HEAD, kv * HEAD, kv * HEAD], 1)
        q, k = _exact_rms(q.unflatten(1, (heads, HEAD)), st["q_norm"]), _exact_rms(k.unflatten(1, (kv, HEAD)), st["k_norm"])
        return _exact_rotated(q, st["table"], st["pos"], HEAD, False), _exact_rotated(k, st["table"], st["pos"], HEAD, False), v.double()
    if kind == "rotary":
        out = []
        for n in "qk":
            v = st[n].double() if st[n + "_norm"] is None else _exact_rms(st[n], st[n + "_norm"])
            out.append(_exact_rotated(v, st["table"], st["pos"], case["part"], case["interleaved"]))
        return tuple(out)
    angle = torch.outer(torch.arange(case["positions"], device=DEV).double(), st["freq"])
    return torch.cat([torch.cos(angle), torch.sin(angle)], 1) * ATTENTION
