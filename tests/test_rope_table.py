"""Angles of stretched contexts by the published rule, which is written in wavelengths, and what rope_table says where a model's factors are not given."""
import math
import warnings

import numpy as np
import pytest

from sapient_b200 import ops
from sapient_b200._lib import SP_ERR_ARG, SapientCudaError


def by_wavelength(f, factor, original, low_freq_factor, high_freq_factor):
    """A frequency whose wavelength is below original / high_freq_factor stays, one above original / low_freq_factor is divided."""
    wavelength = 2 * math.pi / f
    if wavelength < original / high_freq_factor:
        return f
    if wavelength > original / low_freq_factor:
        return f / factor
    smooth = (original / wavelength - low_freq_factor) / (high_freq_factor - low_freq_factor)
    return (1 - smooth) * f / factor + smooth * f


@pytest.mark.parametrize("dim,base,factor,original,low,high", [(128, 500000.0, 8.0, 8192, 1.0, 4.0), (64, 500000.0, 32.0, 8192, 1.0, 4.0), (128, 10000.0, 4.0, 4096, 0.5, 8.0)])
def test_published_rule(dim, base, factor, original, low, high):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        t = ops.rope_table(9000, dim, base, factor=factor, original=original, low=low, high=high)
    f = [by_wavelength(base ** (-2 * i / dim), factor, original, low, high) for i in range(dim // 2)]
    assert any(a == base ** (-2 * i / dim) for i, a in enumerate(f)) and any(a == base ** (-2 * i / dim) / factor for i, a in enumerate(f))
    for p in (1, 17, 4095, 8999):
        want = np.array([[math.cos(p * x), math.sin(p * x)] for x in f])
        # rounded to f32: 2^-25 of 1; the angle in 64 bits: a few roundings of up to 9000
        assert np.abs(t[p] - want).max() <= 2.0**-24


def test_without_a_models_factors_it_warns():
    for given in ({}, {"low": 0.5}, {"high": 4.0}):
        with pytest.warns(UserWarning, match="low_freq_factor"):
            t = ops.rope_table(2, 64, 10000.0, factor=8.0, original=4096, **given)
        assert np.array_equal(t, ops.rope_table(2, 64, 10000.0, factor=8.0, original=4096, low=given.get("low", 0.25), high=given.get("high", 1.0)))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        ops.rope_table(2, 64, 10000.0)
        ops.rope_table(2, 64, 10000.0, factor=4.0)
        assert np.array_equal(ops.rope_table(2, 64, 10000.0, original=4096), ops.rope_table(2, 64, 10000.0))  # nothing is divided by 1


def test_refusals():
    for kw in (dict(original=-1, low=1.0, high=4.0), dict(original=8192, low=4.0, high=1.0), dict(original=8192, low=-1.0, high=4.0), dict(original=8192, low=math.nan, high=4.0)):
        with pytest.raises(SapientCudaError) as e:
            ops.rope_table(3, 4, 10.0, factor=2.0, **kw)
        assert e.value.status == SP_ERR_ARG
