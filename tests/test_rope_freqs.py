"""rope_freqs: the frequencies of every scaling against its definition (CPU)."""

import math

import pytest
import torch


@pytest.fixture(scope="module")
def freqs():
    from pico_hip.kernels import rope_freqs
    return lambda *a, **kw: rope_freqs(*a, device="cpu", **kw)


def test_plain_linear_ntk(freqs):
    f, amp = freqs(64, 1e6)
    assert f.dtype is torch.float64 and amp == 1.0
    want = torch.tensor([1e6 ** (-2 * j / 64) for j in range(32)], dtype=torch.float64)
    assert torch.allclose(f, want, rtol=1e-14, atol=0)
    assert torch.allclose(freqs(64, 1e6, scaling="linear", factor=4.0)[0], want / 4, rtol=1e-14, atol=0)
    # ntk: the slowest pair is slowed by the factor, the fastest not at all
    g = freqs(64, 1e6, scaling="ntk", factor=4.0)[0]
    assert g[0] == 1.0 and math.isclose(float(g[-1]), float(want[-1]) / 4, rel_tol=1e-12)
    factors = [1.0 + j for j in range(32)]
    assert torch.allclose(freqs(64, 1e6, freq_factors=factors)[0], want / torch.tensor(factors), rtol=1e-6, atol=0)


def test_yarn(freqs):
    """Fast pairs stay, slow ones are divided, and the amplitude is 0.1 ln(factor) + 1."""
    plain = freqs(128, 1e6)[0]
    f, amp = freqs(128, 1e6, scaling="yarn", factor=8.0, original_context=32768)
    assert math.isclose(amp, 0.1 * math.log(8.0) + 1)
    turns = 32768 * plain / (2 * math.pi)
    ratio = f / plain
    assert bool((ratio[turns > 33] > 0.95).all()) and float(ratio[0]) == 1.0
    assert torch.allclose(ratio[turns < 0.9], torch.full((), 0.125, dtype=torch.float64))
    assert bool((ratio[1:] <= ratio[:-1] + 1e-15).all())
    assert freqs(128, 1e6, scaling="yarn", factor=0.5, original_context=32768)[1] == 1.0


def test_llama3(freqs):
    plain = freqs(128, 5e5)[0]
    f, amp = freqs(128, 5e5, scaling="llama3", factor=8.0, original_context=8192)
    wave = 2 * math.pi / plain
    for x, y, w in zip(plain.tolist(), f.tolist(), wave.tolist()):
        if w < 8192 / 4:
            want = x
        elif w > 8192:
            want = x / 8
        else:
            s = (8192 / w - 1) / (4 - 1)
            want = (1 - s) * x / 8 + s * x
        assert math.isclose(y, want, rel_tol=1e-12)
    assert amp == 1.0


def test_refusals(freqs):
    for args, kw in [((63,), {}), ((0,), {}), ((64, 0.0), {}), ((64,), dict(scaling="other")),
                     ((64,), dict(scaling="yarn", factor=2.0)), ((64,), dict(scaling="llama3", factor=2.0)),
                     ((64,), dict(factor=0.0)), ((64,), dict(freq_factors=[1.0])), ((2,), dict(scaling="ntk", factor=2.0)),
                     ((64,), dict(scaling="llama3", factor=2.0, original_context=5, low_freq_factor=4.0))]:
        with pytest.raises(ValueError):
            freqs(*args, **kw)
