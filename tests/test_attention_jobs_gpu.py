"""Attention where a launch has two jobs: streams of 33 to 64 rows over a prefix, in blocks of many rows each, and fp32
rows whose blocks are of either kind; and what values that are not finite give the rows that see them.  Tolerances as
in test_attention_gpu.py."""

import pytest
import torch

import aqmi
from test_attention_gpu import TYPES, check_prefix, compare, expected, heads_first, made, off_by_one

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return aqmi.Context(0)


# rows of a stream and key head: 33, 34, 64, 65; 60 with a group of six; 4 of 30 streams, 120 in all; 16 and 17 (fp32's border)
JOBS = [(2, 33, 200, 60, 2, 2, 64), (3, 17, 300, 90, 4, 2, 64), (2, 32, 500, 70, 4, 2, 100), (2, 65, 500, 70, 2, 2, 128),
        (3, 10, 900, 30, 6, 1, 128), (30, 2, 700, 90, 4, 2, 80), (9, 16, 1000, 50, 2, 2, 128), (9, 17, 1000, 50, 2, 2, 128),
        (5, 64, 65, 64, 1, 1, 256), (12, 8, 3000, 700, 4, 2, 64), (8, 4, 129, 33, 12, 3, 33)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lens", [False, True])
@pytest.mark.parametrize("B,T,P,S,H,Hkv,D", JOBS)
def test_two_jobs(ctx, t, lens, B, T, P, S, H, Hkv, D):
    check_prefix(ctx, t, B, T, P, S, H, Hkv, D, lens)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layout", [heads_first, off_by_one])
@pytest.mark.parametrize("B,T,P,S,H,Hkv,D", [JOBS[1], JOBS[5], JOBS[8]])
def test_two_jobs_strides(ctx, t, layout, B, T, P, S, H, Hkv, D):
    check_prefix(ctx, t, B, T, P, S, H, Hkv, D, True, layout)


def causal(q, k, v, pk, pv, b):
    """expected() of a stream whose last T of S keys are its rows' own."""
    T, S, P = q.shape[1], k.shape[1], len(pk)
    sees = torch.cat((torch.ones((T, P), dtype=torch.bool), torch.arange(S) <= S - T + torch.arange(T)[:, None]), 1)
    return expected(q[b], torch.cat((pk, k[b])), torch.cat((pv, v[b])), sees, q.shape[3] ** -0.5)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [64, 100, 128, 256])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("T", [1, 9, 40, 64, 100])
def test_a_value_that_is_not_finite(ctx, t, D, value, T):
    """In a causal key: the rows that see it have that value in its column (scores here are of a few units, so no weight
    vanishes in any type), all else is as without it, bit by bit."""
    g = torch.Generator().manual_seed(T)
    B, P, S, H = 2, 40, T + 13, 2
    q, k, v = made(g, t, B, T, H, D), made(g, t, B, S, H, D), made(g, t, B, S, H, D)
    pk, pv = made(g, t, P, H, D), made(g, t, P, H, D)
    want, got = torch.empty_like(q), torch.empty_like(q)
    aqmi.prefix_attention(ctx, q, pk, pv, k, v, want)
    v[0, 13 + T // 2, 1, 3] = value
    aqmi.prefix_attention(ctx, q, pk, pv, k, v, got)
    want[0, T // 2:, 1, 3] = value
    assert torch.equal(got.nan_to_num(12345.0, float("inf"), float("-inf")), want.nan_to_num(12345.0, float("inf"), float("-inf")))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [64, 100, 256])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("T", [1, 9, 40, 100])
def test_an_infinite_key(ctx, t, D, sign, T):
    """Its score is an infinity of the sign of q's element: -infinity has no weight, +infinity gives NaN, which is what the
    definition gives (exp(infinity - infinity)).  Rows that do not see it are as without it, bit by bit."""
    g = torch.Generator().manual_seed(T)
    B, P, S, H, at = 2, 40, T + 13, 2, 13 + T // 2
    q, k, v = made(g, t, B, T, H, D), made(g, t, B, S, H, D), made(g, t, B, S, H, D, mean=0.25)
    pk, pv = made(g, t, P, H, D), made(g, t, P, H, D, mean=0.25)
    clean, got = torch.empty_like(q), torch.empty_like(q)
    aqmi.prefix_attention(ctx, q, pk, pv, k, v, clean)
    k[0, at, 1, 3] = sign * float("inf")
    aqmi.prefix_attention(ctx, q, pk, pv, k, v, got)
    up = q[0, T // 2:, 1, 3] * sign > 0
    later = got[0, T // 2:, 1]
    assert later[up].isnan().all()
    rest = torch.ones((B, T, H), dtype=torch.bool, device="cuda")
    rest[0, T // 2:, 1] = False
    assert torch.equal(got[rest], clean[rest])
    # The others as without that key: expected() of the rows that see it, of head 1, with the key taken out.
    kept = [j for j in range(S) if j != at]
    parts = causal(q[:, T // 2:, 1:], k[:, kept, 1:], v[:, kept, 1:], pk[:, 1:], pv[:, 1:], 0) if T // 2 < T else None
    down = (~up).nonzero()[:, 0].cpu()
    if len(down):
        compare([later[down.cuda()][:, None]], [tuple(p[down] for p in parts)], t)
