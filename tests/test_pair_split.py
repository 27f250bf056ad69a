"""The bounds that two scaled fp16 numbers of an fp32 value keep, by the arithmetic of the split itself: h is the nearest fp16
number, l the nearest of 2^11 times what is left."""
import numpy as np
import pytest


def _split(x, largest):
    v = np.ldexp(x.astype(np.float32), 15 - int(np.frexp(np.float32(largest))[1]))   # the largest comes into [2^14, 2^15)
    h = v.astype(np.float16)
    rest = v - h.astype(np.float32)   # exact
    l = (rest * np.float32(2 ** 11)).astype(np.float16)
    return v.astype(np.float64), h.astype(np.float64), l.astype(np.float64) * 2.0 ** -11


@pytest.mark.parametrize("largest", [1.0, 1.5, 2 - 2.0 ** -23, 2.0 ** 40, 2.0 ** -140])
@pytest.mark.parametrize("power", [0, 3, 11, 16, 17, 24, 26, 27])
def test_elements_within_2_to_the_27(largest, power):
    rng = np.random.RandomState(power)
    x = (largest * 2.0 ** -power * np.concatenate([rng.uniform(1, 2, 20000), 1 + 2.0 ** -np.arange(1.0, 24)])).astype(np.float32)
    x = np.minimum(x, np.float32(largest))
    v, h, l = _split(x, largest)
    assert np.isfinite(h).all()
    assert (np.abs(l) <= 2.0 ** -11 * np.abs(v)).all()          # what a product of two such is left off by is 2^-22 of it
    assert (np.abs(v - h - l) <= 2.0 ** -23 * np.abs(v)).all()


@pytest.mark.parametrize("power", list(range(28, 60)))
def test_smaller_elements(power):
    x = (2.0 ** -power * np.random.RandomState(power).uniform(1, 2, 20000)).astype(np.float32)
    for largest in (1.0, 2 - 2.0 ** -23):
        v, h, l = _split(x, largest)
        assert (np.abs(v - h - l) <= 2.0 ** -36).all()   # 2^-50 of the largest value, which is 2^14 or more here
