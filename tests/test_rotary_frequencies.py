"""rotary_frequencies and Rotary: the published formulas, and what is refused."""
import math

import numpy as np
import pytest
import torch

from kunserve_amd import Rotary, rotary_frequencies

N = 128


def test_plain_and_linear():
    f, scale = rotary_frequencies(N, 10000.0)
    assert scale == 1.0 and f.dtype == np.float64
    for j in (0, 1, 17, 63):
        assert f[j] == pytest.approx(10000.0 ** (-2 * j / N), rel=1e-14)
    for kind in ("default", "linear"):
        g, scale = rotary_frequencies(N, 10000.0, dict(rope_type=kind, factor=4.0))
        assert scale == 1.0
        np.testing.assert_allclose(g, f / (4 if kind == "linear" else 1), rtol=1e-15)


def test_ntk_keeps_the_fastest_and_slows_the_slowest_by_the_factor():
    f, _ = rotary_frequencies(N, 10000.0)
    g, _ = rotary_frequencies(N, 10000.0, dict(type="ntk", factor=8.0))
    assert g[0] == 1.0
    assert g[-1] == pytest.approx(f[-1] / 8, rel=1e-13)
    assert np.all(np.diff(g / f) < 0)
    # nothing to slow in a single pair
    np.testing.assert_array_equal(rotary_frequencies(2, 1e4, dict(type="ntk", factor=8.0))[0], [1.0])


def test_llama3_by_wavelength():
    """Wavelengths below length / high keep their frequency, those above length /
    low are divided, between the two by the published interpolation."""
    sc = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
              original_max_position_embeddings=8192)
    f, _ = rotary_frequencies(N, 500000.0)
    g, scale = rotary_frequencies(N, 500000.0, sc)
    assert scale == 1.0
    kinds = set()
    for a, b in zip(f, g):
        wave = 2 * math.pi / a
        if wave < 8192 / 4.0:
            want, kind = a, "kept"
        elif wave > 8192 / 1.0:
            want, kind = a / 8, "slowed"
        else:
            smooth = (8192 / wave - 1.0) / (4.0 - 1.0)
            want, kind = (1 - smooth) * a / 8 + smooth * a, "between"
        kinds.add(kind)
        assert b == pytest.approx(want, rel=1e-13)
    assert kinds == {"kept", "slowed", "between"}


def test_yarn_ramp_and_attention_factor():
    sc = dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096)
    f, _ = rotary_frequencies(N, 10000.0)
    g, scale = rotary_frequencies(N, 10000.0, sc)
    assert scale == pytest.approx(0.1 * math.log(16) + 1, rel=1e-15)
    turns = lambda j: 4096 * 10000.0 ** (-2 * j / N) / (2 * math.pi)   # noqa: E731
    first = max(j for j in range(N // 2) if turns(j) >= 32)
    last = min(j for j in range(N // 2) if turns(j) <= 1)
    for j in range(N // 2):
        slowed = min(max((j - first) / (last - first), 0), 1)
        assert g[j] == pytest.approx(f[j] * (1 - slowed) + f[j] / 16 * slowed, rel=1e-13)
    assert rotary_frequencies(N, 1e4, dict(sc, attention_factor=2.5))[1] == 2.5
    np.testing.assert_array_equal(
        rotary_frequencies(N, 1e4, dict(sc, beta_fast=32, beta_slow=1))[0], g)


@pytest.mark.parametrize("args,what", [
    ((0,), "rotary_dim"), ((7,), "rotary_dim"), ((64, 0.0), "theta"), ((64, float("nan")), "theta"),
    ((64, 1e4, dict(rope_type="other")), "rope_type"), ((64, 1e4, {}), "rope_type"),
    ((64, 1e4, dict(rope_type="linear", factor=0.5)), "factor"),
    ((64, 1e4, dict(rope_type="linear", factor=float("inf"))), "factor"),
    ((64, 1e4, dict(rope_type="yarn", factor=2.0)), "original_max"),
    ((64, 1e4, dict(rope_type="llama3", factor=2.0, original_max_position_embeddings=0)),
     "original_max"),
    ((64, 1e4, dict(rope_type="llama3", factor=2.0, original_max_position_embeddings=100,
                    low_freq_factor=4.0, high_freq_factor=4.0)), "low_freq_factor"),
    ((64, 1e4, dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=100,
                    beta_fast=1.0, beta_slow=1.0)), "beta_slow"),
    ((64, 1.0, dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=100)), "theta"),
])
def test_refused_frequencies(args, what):
    with pytest.raises(ValueError, match=what):
        rotary_frequencies(*args)


def test_rotary_object():
    r = Rotary(64, 1e4, device="cpu", scaling=dict(rope_type="yarn", factor=4.0,
                                                   original_max_position_embeddings=2048))
    assert r.frequencies.dtype == torch.float64 and r.frequencies.shape == (32,)
    assert r.scale == pytest.approx(0.1 * math.log(4) + 1)
    own = Rotary(32, frequencies=np.linspace(1, 0.1, 16), scale=1.5, device="cpu")
    assert own.scale == 1.5 and float(own.frequencies[-1]) == pytest.approx(0.1)
    for kw, what in ((dict(rotary_dim=24), "multiple of 16"), (dict(rotary_dim=0), "multiple of 16"),
                     (dict(rotary_dim=32, frequencies=np.ones(15)), "finite frequencies"),
                     (dict(rotary_dim=32, frequencies=np.full(16, np.nan)), "finite frequencies"),
                     (dict(rotary_dim=32, frequencies=np.ones(16),
                           scaling=dict(rope_type="linear", factor=2.0)), "no meaning"),
                     (dict(rotary_dim=32, scale=float("inf")), "not finite")):
        with pytest.raises(ValueError, match=what):
            Rotary(device="cpu", **kw)
    with pytest.raises(ValueError, match="exceeds"):
        r.check(32, torch.device("cpu"))
    with pytest.raises(ValueError, match="frequencies are on"):
        r.check(64, torch.device("meta"))
