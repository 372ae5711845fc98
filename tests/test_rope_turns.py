"""CPU tests of rope_turns' blend between kept and divided frequencies."""

import math

import numpy as np
import pytest

from turboquant.core.rope import rope_turns


def by_parts(**kw):
    return rope_turns(**{**dict(rotary_dim=128, theta=1e6, scaling="by_parts", factor=4.0, trained_length=32768), **kw})


def test_blend_by_index():
    """Pairs turn 32 times at index 23.6 and once at 39.7: kept up to 23, a quarter from 40 on, linear in between."""
    plain = rope_turns(128, theta=1e6)[0].numpy()
    assert plain[23] * 32768 > 32 > plain[24] * 32768 and plain[39] * 32768 > 1 > plain[40] * 32768
    got, mag = by_parts(blend="index")
    share = np.clip((40 - np.arange(64)) / 17, 0, 1)
    np.testing.assert_allclose(got.numpy(), plain * (share + (1 - share) / 4), rtol=1e-14)
    assert mag == pytest.approx(0.1 * math.log(4) + 1)
    turns, _ = by_parts()
    assert np.array_equal(turns.numpy(), by_parts(blend="turns")[0].numpy())
    ends = (np.arange(64) <= 23) | (np.arange(64) >= 40)
    np.testing.assert_allclose(turns.numpy()[ends], got.numpy()[ends], rtol=1e-14)
    assert turns[32] / got[32] == pytest.approx(0.584, abs=5e-4)


def test_blend_at_the_ends():
    """Lengths over which no pair turns `fast` times, none turns `slow` times, and all do."""
    plain = rope_turns(64, theta=500.0)[0].numpy()
    few = by_parts(rotary_dim=64, theta=500.0, trained_length=100, blend="index")[0].numpy()
    n = plain * 100
    assert n[0] < 32 and few[0] == pytest.approx(plain[0], rel=1e-14) and np.allclose(few[n <= 1], plain[n <= 1] / 4, rtol=1e-14)
    assert np.all(few <= plain * (1 + 1e-14)) and np.all(few >= plain / 4 * (1 - 1e-14))
    none = by_parts(rotary_dim=64, theta=500.0, trained_length=3, blend="index")[0].numpy()
    np.testing.assert_allclose(none, plain / 4, rtol=1e-14)
    every = by_parts(rotary_dim=64, theta=500.0, trained_length=10 ** 7, blend="index")[0].numpy()
    np.testing.assert_allclose(every, plain, rtol=1e-14)
    for kw in (dict(blend="x"), dict(blend="index", theta=1.0), dict(blend="index", slow=0.0)):
        with pytest.raises(ValueError):
            by_parts(**kw)
