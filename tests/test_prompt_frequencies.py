"""Frequencies of position rotations: arguments that a scaling does not name are
not looked at, whatever they hold."""
import ctypes
import math

import numpy as np
import pytest

import mlxcel_amd as mq
from mlxcel_amd import _lib

NAN, INF = math.nan, math.inf
UNUSED = (0.0, -1.0, NAN, INF, -INF)
PLAIN, LINEAR, BASE, BANDS, RAMP = range(5)


def frequencies(dims, base, scaling, factor, original, low, high):
    lib = _lib.load()
    inv, by = (ctypes.c_float * (dims // 2))(), ctypes.c_float(-1.0)
    assert lib.mlxq_rotary_frequencies(dims, base, scaling, factor, original, low, high, inv, ctypes.byref(by)) == 0
    return np.array(inv), by.value


@pytest.mark.parametrize("x", UNUSED)
def test_plain_looks_at_no_factor(x):
    want, by = frequencies(8, 10000.0, PLAIN, 1.0, 1.0, 1.0, 4.0)
    np.testing.assert_allclose(want, 10000.0 ** (-np.arange(0, 8, 2) / 8), rtol=2.0 ** -23)
    assert by == 1
    for args in ((x, 1.0, 1.0, 4.0), (1.0, x, x, x), (x, x, x, x)):
        got, by = frequencies(8, 10000.0, PLAIN, *args)
        assert np.array_equal(got, want) and by == 1, args
    got, by = mq.rotary_frequencies(8, factor=x, original=x, low=x, high=x, device="cpu")
    assert np.array_equal(got.numpy(), want) and by == 1


@pytest.mark.parametrize("scaling", [LINEAR, BASE])
@pytest.mark.parametrize("x", UNUSED)
def test_linear_and_base_look_at_no_lengths(scaling, x):
    want, _ = frequencies(8, 10000.0, scaling, 4.0, 1.0, 1.0, 4.0)
    assert np.isfinite(want).all()
    got, by = frequencies(8, 10000.0, scaling, 4.0, x, x, x)
    assert np.array_equal(got, want) and by == 1


@pytest.mark.parametrize("scaling", [LINEAR, BASE, BANDS, RAMP])
@pytest.mark.parametrize("factor", [0.0, 0.5, -1.0, NAN, INF])
def test_a_factor_that_is_used_is_refused(scaling, factor):
    inv, by = (ctypes.c_float * 4)(), ctypes.c_float()
    assert _lib.load().mlxq_rotary_frequencies(8, 1e4, scaling, factor, 100.0, 1.0, 4.0, inv, ctypes.byref(by)) == _lib.EINVAL
