"""A configuration's scaling is taken whole: each key that changes frequencies or
factor does so here, and what is not understood raises."""
import math

import numpy as np
import pytest

from kunserve_amd import Rotary, rotary_frequencies

YARN = dict(rope_type="yarn", factor=32.0, original_max_position_embeddings=4096,
            beta_fast=32.0, beta_slow=1.0)


def ramp(n, theta, length, fast, slow, rounded):
    """The share of f / factor in each pair's frequency, from the turns of the pairs
    (real numbers) that the ramp begins and ends at."""
    at = lambda turns: n * math.log(length / (2 * math.pi * turns)) / (2 * math.log(theta))   # noqa: E731
    lo, hi = at(fast), at(slow)
    if rounded:
        lo, hi = math.floor(lo), math.ceil(hi)
    return np.array([min(max((j - lo) / (hi - lo), 0.0), 1.0) for j in range(n // 2)])


@pytest.mark.parametrize("truncate", [True, False, None])
@pytest.mark.parametrize("n,theta", [(64, 150000.0), (128, 10000.0)])
def test_yarn_ramp_ends(n, theta, truncate):
    f, _ = rotary_frequencies(n, theta)
    g, scale = rotary_frequencies(n, theta, dict(YARN, truncate=truncate))
    s = ramp(n, theta, 4096, 32.0, 1.0, truncate is not False)
    np.testing.assert_allclose(g, f * (1 - s) + f / 32.0 * s, rtol=1e-12)
    assert scale == pytest.approx(0.1 * math.log(32.0) + 1, rel=1e-15)


def test_truncate_matters():
    a, b = (rotary_frequencies(64, 150000.0, dict(YARN, truncate=x))[0] for x in (True, False))
    assert np.max(np.abs(a / b - 1)) > 0.5


@pytest.mark.parametrize("m,m_all", [(1.0, 1.0), (0.707, 0.707), (1.0, 0.5), (0.25, 2.0)])
def test_yarn_mscale(m, m_all):
    _, scale = rotary_frequencies(64, 1e4, dict(YARN, factor=40.0, mscale=m, mscale_all_dim=m_all))
    want = (0.1 * m * math.log(40.0) + 1) / (0.1 * m_all * math.log(40.0) + 1)
    assert scale == pytest.approx(want, rel=1e-15)
    given = dict(YARN, mscale=m, mscale_all_dim=m_all, attention_factor=1.25)
    assert Rotary(64, 1e4, scaling=given, device="cpu").scale == 1.25


@pytest.mark.parametrize("scaling,what", [
    (dict(YARN, mscale=1.0), "given together"), (dict(YARN, mscale_all_dim=0.7), "given together"),
    (dict(YARN, mscale=0.0, mscale_all_dim=0.0), "positive"),
    (dict(YARN, mscale=math.nan, mscale_all_dim=1.0), "positive"),
    (dict(YARN, truncate="no"), "truncate"),
    (dict(YARN, attention_factor=math.inf), "attention_factor"),
    (dict(YARN, low_freq_factor=1.0), "'low_freq_factor'"),
    (dict(YARN, long_factor=[1.0], short_factor=[1.0]), "'long_factor', 'short_factor'"),
    (dict(YARN, partial_rotary_factor=0.5), "'partial_rotary_factor'"),
    (dict(YARN, rope_theta=1e6), "rope_theta"),
    (dict(YARN, type="linear"), "differ"),
    (dict(YARN, factor=None), "needs a factor"),
    (dict(rope_type="linear"), "needs a factor"), (dict(rope_type="ntk"), "needs a factor"),
    (dict(rope_type="llama3", original_max_position_embeddings=8192), "needs a factor"),
    (dict(rope_type="linear", factor=2.0, attention_factor=1.0), "'attention_factor'"),
    (dict(rope_type="llama3", factor=8.0, original_max_position_embeddings=8192, beta_fast=32.0),
     "'beta_fast'"),
    (dict(rope_type="default", mrope_section=[16, 24, 24]), "'mrope_section'"),
])
def test_keys_that_are_not_understood(scaling, what):
    with pytest.raises(ValueError, match=what):
        rotary_frequencies(64, 1e4, scaling)


def test_keys_that_change_nothing():
    f, _ = rotary_frequencies(64, 1e4, dict(rope_type="linear", factor=2.0))
    for more in (dict(original_max_position_embeddings=2048), dict(rope_theta=10000),
                 dict(attention_factor=None), dict(type="linear")):
        np.testing.assert_array_equal(
            rotary_frequencies(64, 1e4, dict(rope_type="linear", factor=2.0, **more))[0], f)
