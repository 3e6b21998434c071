"""tle_rope_frequencies, every pair against the definition (tests/test_cache8_abi.py
has its refusals and the ends): contexts for which no pair turns less than once, few or all do.
"""
import numpy as np
import pytest

import tle


def yarn(d, base, factor, ctx):
    """Frequencies by counting turns: the ramp goes from the last pair of at least 32 turns (or pair 0) to the
    first one of at most one turn, both looked for among as many pairs as it takes."""
    turns = lambda i: ctx * float(base) ** (-2.0 * i / d) / (2 * np.pi)  # noqa: E731
    lo = 0
    while turns(lo + 1) >= 32:
        lo += 1
    hi = 0
    while turns(hi) > 1:
        hi += 1
    f = float(base) ** (-2.0 * np.arange(d // 2) / d)
    i = np.arange(d // 2)
    slow = np.where(i >= hi, 1.0, np.where(i <= lo, 0.0, (i - lo) / max(hi - lo, 1)))
    return f * (1 - slow) + f / factor * slow


@pytest.mark.parametrize("d", [16, 32, 48, 64])
@pytest.mark.parametrize("base", [10000.0, 500000.0, 100.0])
@pytest.mark.parametrize("ctx", [1, 6, 7, 150, 2048, 4096, 32768, 40960, 131072, 1 << 20, 1 << 30])
def test_yarn_at_every_pair(d, base, ctx):
    for factor in (1.0, 4.0, 40.0):
        f, m = tle.rope_frequencies(d, base, "yarn", factor, ctx)
        want = yarn(d, base, factor, ctx)
        # one rounding to 32 bits, and 64-bit powers
        assert np.all(np.abs(np.array(f) - want) <= want * (2.0 ** -24 + 2.0 ** -45)), (f, want)
        assert abs(m - (1 + 0.1 * np.log(factor))) <= m * (2.0 ** -24 + 2.0 ** -45)
        turns = ctx * base ** (-2.0 * np.arange(d // 2) / d) / (2 * np.pi)
        plain = base ** (-2.0 * np.arange(d // 2) / d)
        assert np.allclose(np.array(f)[turns > 32], plain[turns > 32], rtol=2.0 ** -23, atol=0)
        assert np.allclose(np.array(f)[turns < 1], plain[turns < 1] / factor, rtol=2.0 ** -23, atol=0)


def test_a_slow_last_pair_keeps_its_place_in_the_ramp():
    """The last pair turns 2.8 times within 131072 rows: 0.69 of the way, not all of it."""
    f, _ = tle.rope_frequencies(64, 10000.0, "yarn", 4.0, 131072)
    plain = 10000.0 ** (-62 / 64)
    assert abs(f[-1] / plain - (1 - 9 / 13 * 0.75)) <= 1e-6
