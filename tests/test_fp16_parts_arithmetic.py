"""The two fp16 parts of the gated feed-forward block's large products, in NumPy: how
far a value may be off, with exponents of rows and of blocks, and that taking a
block's parts to another exponent rounds no h."""
import numpy as np
import pytest

from tests.helpers import rng

DOWN = 4   # blocks: as many powers of two that h may be divided by


def split(v, down):
    """Parts h, l of scaled values, |v| < 2^15: v = h + l / 2^11 but for rounding."""
    h = np.float16(np.float32(np.float16(v * np.float32(2.0 ** -down))) * np.float32(2.0 ** down))
    l = np.float16((v - np.float32(h)) * np.float32(2048))
    return h, l


def values(seed):
    """Of all sizes below 2^15, those next to powers of two among them."""
    r = rng(seed)
    v = np.float32(r.uniform(-1, 1, 200_000) * 2.0 ** r.integers(-60, 16, 200_000))
    p = np.float32(2.0 ** np.arange(-60, 15))
    return np.concatenate([v, p, -p, np.nextafter(p, np.float32(0)), np.nextafter(p, np.float32(np.inf)),
                           np.nextafter(np.float32(2 ** 15), np.float32(0), dtype=np.float32)[None], np.zeros(1, np.float32)])


@pytest.mark.parametrize("down", [0, DOWN])
def test_a_value_is_off_by_no_more(down):
    v = values(1)
    h, l = split(v, down)
    assert np.isfinite(h).all() and np.isfinite(l).all()
    off = np.abs(v.astype(np.float64) - (h.astype(np.float64) + l.astype(np.float64) / 2048))
    assert (off <= np.maximum(2.0 ** -23 * np.abs(v.astype(np.float64)), 2.0 ** (-36 if down == 0 else -33))).all()


@pytest.mark.parametrize("down", [0, DOWN])
def test_the_small_part_is_no_larger(down):
    """|l| <= |h|, but for what small values leave, 2^(down - 14)."""
    v = values(2)
    h, l = (p.astype(np.float64) for p in split(v, down))
    assert (np.abs(l) <= np.maximum(np.abs(h), 2.0 ** (down - 14))).all()


@pytest.mark.parametrize("d", range(DOWN + 1))
def test_the_large_part_goes_to_another_exponent_unrounded(d):
    h, l = split(values(3), DOWN)
    by = np.float16(2.0 ** -d)
    assert ((h * by).astype(np.float64) == h.astype(np.float64) * 2.0 ** -d).all()
    off = np.abs((l * by).astype(np.float64) - l.astype(np.float64) * 2.0 ** -d)
    assert off.max() <= 2.0 ** -25   # 2^-36 of a value
