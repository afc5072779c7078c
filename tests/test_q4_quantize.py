"""q4_quantize on the host: codes within half a step, and what it refuses."""

import numpy as np
import pytest

import aqmi


def dense(codes, scale, zero, K, G):
    q = np.stack((codes & 15, codes >> 4), 2).reshape(len(codes), -1)[:, :K].astype(np.float64)
    at = np.arange(K) // G
    return (q - (8 if zero is None else zero.astype(np.float64)[:, at])) * scale.astype(np.float64)[:, at]


@pytest.mark.parametrize("K,G", [(1, 32), (33, 32), (100, 64), (256, 128)])
@pytest.mark.parametrize("zeros", [False, True])
def test_codes_are_the_nearest(K, G, zeros):
    w = np.random.default_rng(K).standard_normal((7, K)).astype(np.float32)
    w[3] = 0
    codes, scale, zero = aqmi.q4_quantize(w, G, zeros)
    assert codes.shape == (7, (K + 1) // 2) and scale.shape == (7, -(-K // G)) and (zero is not None) == zeros
    step = np.repeat(scale.astype(np.float64), G, 1)[:, :K]
    # Half a step; the scale's rounding to 11 bits moves the ends (7 or 15
    # steps out) by 15 * 2^-12, and a zero's own rounding by half a step more.
    assert np.all(np.abs(dense(codes, scale, zero, K, G) - w) <= (0.5 + 15 * 2.0 ** -11 + (0.5 if zeros else 0)) * step + 1e-12)
