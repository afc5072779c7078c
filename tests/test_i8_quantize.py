"""aqmi.i8_quantize: a matrix in 8 bits with a scale for each row, on the host."""

import numpy as np
import pytest

import aqmi


@pytest.mark.parametrize("N,K", [(1, 1), (3, 7), (40, 129)])
def test_half_a_step(N, K):
    w = np.random.default_rng(N).standard_normal((N, K)).astype(np.float32)
    codes, scale = aqmi.i8_quantize(w)
    assert codes.dtype == np.int8 and scale.dtype == np.float32 and codes.shape == w.shape and scale.shape == (N,)
    # half a step of the unrounded scale, and the scale's own rounding times up to 127
    assert np.all(np.abs(codes * scale.astype(np.float64)[:, None] - w) <= (0.5 + 127 * 2.0 ** -24 + 1e-9) * scale[:, None])
    assert np.all(np.abs(codes).max(1) == 127)


def test_rows_of_zeros():
    codes, scale = aqmi.i8_quantize(np.zeros((2, 5), np.float32))
    assert not codes.any() and not scale.any()


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_refuses_what_is_not_finite(value):
    w = np.ones((3, 4), np.float32)
    w[1, 2] = value
    with pytest.raises(ValueError, match="row 1"):
        aqmi.i8_quantize(w)
