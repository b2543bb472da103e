"""CPU tests of the rotary layer: the scaled frequencies against their
formulas, and refusals."""

import math

import pytest
import torch

from minisgl_amd.layers import RotaryEmbedding, rotary_frequencies


def test_default_and_linear():
    f, s = rotary_frequencies(8, 10000.0)
    assert s == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    g, _ = rotary_frequencies(8, 10000.0, {"type": "linear", "factor": 4.0})
    assert torch.equal(g, f / 4)


def test_dynamic():
    scaling = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 1000}
    same, _ = rotary_frequencies(64, 1e4, scaling, 500)
    assert torch.allclose(same, rotary_frequencies(64, 1e4)[0], rtol=1e-13)
    f, s = rotary_frequencies(64, 1e4, scaling, 4000)
    base = 1e4 * (2.0 * 4 - 1) ** (64 / 62)
    assert s == 1.0 and torch.allclose(f, rotary_frequencies(64, base)[0], rtol=1e-13)


def test_llama3():
    scaling = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": 8192}
    f, s = rotary_frequencies(128, 5e5, scaling)
    plain = rotary_frequencies(128, 5e5)[0]
    assert s == 1.0
    for a, b in zip(f.tolist(), plain.tolist()):
        wave = 2 * math.pi / b
        if wave < 8192 / 4:
            want = b
        elif wave > 8192 / 1:
            want = b / 8
        else:
            t = (8192 / wave - 1) / 3
            want = (1 - t) * b / 8 + t * b
        assert a == pytest.approx(want, rel=1e-13)


def test_yarn():
    scaling = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    f, s = rotary_frequencies(128, 1e6, scaling)
    plain = rotary_frequencies(128, 1e6)[0]
    assert s == pytest.approx(0.1 * math.log(4) + 1)
    # turns over the original context: kept above 32, divided below 1
    turns = 32768 * plain / (2 * math.pi)
    assert torch.equal(f[turns > 40], plain[turns > 40])
    assert torch.allclose(f[turns < 0.8], plain[turns < 0.8] / 4, rtol=1e-13)
    mid = (turns < 30) & (turns > 1.2)
    assert ((f < plain) & (f > plain / 4))[mid].all()
    assert rotary_frequencies(128, 1e6, {**scaling, "attention_factor": 1.5})[1] == 1.5
    both = rotary_frequencies(128, 1e6, {**scaling, "mscale": 0.7, "mscale_all_dim": 1.0})[1]
    assert both == pytest.approx((0.07 * math.log(4) + 1) / (0.1 * math.log(4) + 1))


@pytest.mark.parametrize("call", [
    lambda: rotary_frequencies(7, 1e4),
    lambda: rotary_frequencies(0, 1e4),
    lambda: rotary_frequencies(8, 1e4, {"type": "longrope"}),
    lambda: rotary_frequencies(8, 1e4, {"type": "linear"}),
    lambda: rotary_frequencies(8, 1e4, {"type": "linear", "factor": 0}),
    lambda: rotary_frequencies(8, 1e4, {"type": "yarn", "factor": 4.0}),
    lambda: rotary_frequencies(8, 1e4, {"type": "llama3", "factor": 4.0, "original_max_position_embeddings": 8, "low_freq_factor": 4,
                                        "high_freq_factor": 4}),
    lambda: RotaryEmbedding(64, 128, 10, 1e4),
    lambda: RotaryEmbedding(64, 64, 0, 1e4),
    lambda: RotaryEmbedding(64, 64, 8, 1e4).forward(torch.arange(2), torch.zeros(2, 64), torch.zeros(2, 64)),
])
def test_refusals(call):
    with pytest.raises(ValueError):
        call()


def test_layer_has_no_state():
    assert RotaryEmbedding(64, 64, 8, 1e4).state_dict() == {}


def test_yarn_without_truncation():
    """The ramp between the real-valued indices whose waves turn beta_fast
    and beta_slow times over the original context."""
    d, base, original, factor = 64, 1.5e5, 4096, 32.0
    f, _ = rotary_frequencies(d, base, {"rope_type": "yarn", "factor": factor, "beta_fast": 32.0, "beta_slow": 1.0,
                                        "original_max_position_embeddings": original, "truncate": False})
    low, high = (d * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base)) for turns in (32.0, 1.0))
    for i, got in enumerate(f.tolist()):
        plain = base ** (-2 * i / d)
        t = min(max((i - low) / (high - low), 0.0), 1.0)
        assert got == pytest.approx(plain * (1 - t) + plain / factor * t, rel=1e-12)


@pytest.mark.parametrize("base", [1.0, 0.0, -10000.0, float("nan")])
def test_base_refused(base):
    with pytest.raises(ValueError, match="base"):
        rotary_frequencies(8, base)


def test_prepare_refuses_the_cpu():
    with pytest.raises(ValueError, match="GPU"):
        RotaryEmbedding(64, 64, 8, 1e4).prepare(torch.device("cpu"))
