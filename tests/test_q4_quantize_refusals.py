"""What q4_quantize refuses: weights without a finite float16 scale, whose
products would not be finite either."""

import numpy as np
import pytest

import aqmi


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 2e6, -2e6, 3e38])
def test_no_finite_scale(zeros, bad):
    w = np.random.default_rng(1).standard_normal((5, 100)).astype(np.float32)
    w[3, 70] = bad
    with pytest.raises(ValueError, match="row 3, columns from 64"):
        aqmi.q4_quantize(w, 64, zeros)


@pytest.mark.parametrize("zeros,most", [(False, 65504 * 7), (True, 65504 * 15)])
def test_the_largest_that_has_one(zeros, most):
    w = np.zeros((1, 32), np.float32)
    w[0, 5] = most
    codes, scale, zero = aqmi.q4_quantize(w, 32, zeros)
    assert scale[0, 0] == 65504 and codes[0, 2] >> 4 == 15
