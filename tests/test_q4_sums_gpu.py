"""The sums of aq_q4_forward for rows of x with a mean, against 64 bits.

The codes enter as 16 + q and the offset is taken off the group's sum, so for
x of one sign that sum is many times its result, and what is rounded at its
size shows.  For x in [1, 2] nothing is rounded there.  A floating x (of an
fp32 one the upper 8 bits of the mantissa) then lies on one grid, 2^-10 for
f16 and 2^-7 for bf16: with at most 128 columns and factors up to 31 its sums
are at most 2^13, 23 bits on that grid, and exact, as is the offset's part of
them.  The other 16 bits of an fp32 x are below 2^-7 of it, and so are the
roundings of their sums beside what the upper part's would be.  What is left
is a rounding of each group's scaled sum, of the running sum, and of the sum
of each wave's part: 2^-24 at most of values no larger, in the norm, than the
result.  With at most 32 groups and 8 waves and random signs that is
sqrt(2 * 32 + 8) * 2^-24 / sqrt(3) = 2.9e-7; 4e-7 is asked.  Whole numbers are
exact up to the scaling, one rounding more at the end."""

import numpy as np
import pytest
import torch

import aqmi

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8,
         "e4m3": torch.float8_e4m3fn}


@pytest.fixture(scope="module")
def ctx():
    return aqmi.Context(0)


def matrix(N, K, G, seed):
    r = np.random.default_rng(seed)
    shape = (N, -(-K // G))
    codes = r.integers(0, 256, (N, (K + 1) // 2), dtype=np.uint8)
    scale = (r.uniform(0.5, 1.5, shape) / np.sqrt(K)).astype(np.float16)
    zero = r.integers(0, 16, shape, dtype=np.uint8)
    q = np.stack((codes & 15, codes >> 4), 2).reshape(N, -1)[:, :K].astype(np.float64)
    at = np.arange(K) // G
    return codes, scale, zero, (q - zero.astype(np.float64)[:, at]) * scale.astype(np.float64)[:, at]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("N,K,M", [(515, 1000, 5), (515, 1000, 64), (515, 1024, 33), (9000, 1024, 3), (26000, 1024, 16)])
def test_rows_with_a_mean(ctx, t, G, N, K, M):
    codes, scale, zero, w = matrix(N, K, G, N + K + G)
    lin = aqmi.Q4Linear(ctx, codes, scale, K, G, zero)
    x = 1 + torch.rand(M, K, generator=torch.Generator().manual_seed(M))
    s = None
    if t in ("i8", "e4m3"):
        x = (63 * x).round()   # 63 .. 126
        s = torch.full((M, 1), 1 / 64.0, device="cuda")
    x = x.to(TYPES[t])
    y = torch.empty((M, N), device="cuda")
    lin.forward(x.cuda(), y, s)
    ref = x.double().numpy() / (1 if s is None else 64) @ w.T
    assert np.linalg.norm(y.double().cpu().numpy() - ref) <= 4e-7 * np.linalg.norm(ref)
