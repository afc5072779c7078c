"""Calls that the operators split: more rows of x than one packed batch of a
4-bit product holds, more long rows than one group of a sampling call, and
rows near the longest that it takes.

A product's tolerance is that of tests/test_q4_gpu.py: 2e-6 of the result's
norm.  A wave adds some 200 groups one after another here, which for random
signs is sqrt(200) * 2^-24 / sqrt(3) = 4.9e-7 of it.  Sampling is held to the
whole-number reference of tests/test_sample_gpu.py, token for token."""

import numpy as np
import pytest
import torch
from test_sample_gpu import check, normal

import aqmi

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8,
         "e4m3": torch.float8_e4m3fn}


@pytest.fixture(scope="module")
def ctx():
    return aqmi.Context(0)


# A packed row takes 768 bytes a block of 128 columns in fp32, 256 in the other
# types and 128 in int8; a batch is 64 MB in whole 64 rows: 640 rows each time.
@pytest.mark.parametrize("t,K", [("f32", 16000), ("f16", 50000), ("bf16", 50001), ("i8", 100000), ("e4m3", 50000)])
@pytest.mark.parametrize("M", [640, 641, 1300])
def test_rows_of_several_batches(ctx, t, K, M):
    N, G, xg = 20, 128, 64 if t in ("i8", "e4m3") else 0
    r = np.random.default_rng(K + M)
    codes = r.integers(0, 256, (N, (K + 1) // 2), dtype=np.uint8)
    scale = (r.uniform(0.5, 1.5, (N, -(-K // G))) / np.sqrt(K)).astype(np.float16)
    zero = r.integers(0, 16, scale.shape, dtype=np.uint8)
    bias = r.standard_normal(N).astype(np.float32)
    lin = aqmi.Q4Linear(ctx, codes, scale, K, G, zero, bias)
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn((M, K), generator=g, device="cuda")
    s = None
    if xg:
        x = (x * 30).clamp(-127, 127).round()
        s = torch.rand((M, -(-K // xg)), generator=g, device="cuda") + 0.5
    x = x.to(TYPES[t])
    y = torch.full((M, N + 3), 7.0, device="cuda")
    lin.forward(x, y[:, :N], s, xg)
    q = np.stack((codes & 15, codes >> 4), 2).reshape(N, -1)[:, :K].astype(np.float64)
    at = np.arange(K) // G
    w = torch.from_numpy((q - zero.astype(np.float64)[:, at]) * scale.astype(np.float64)[:, at]).cuda()
    for m in range(0, M, 640):   # each batch for itself
        xd = x[m:m + 640].double()
        if xg:
            xd = xd * s[m:m + 640].double().repeat_interleave(xg, 1)[:, :K]
        ref = torch.mm(w, xd.t().contiguous()).t() + torch.from_numpy(bias).cuda().double()
        assert float((y[m:m + 640, :N].double() - ref).norm()) <= 2e-6 * float(ref.norm())
    assert bool((y[:, N:] == 7).all())


@pytest.mark.parametrize("rows", [256, 257, 530])
def test_long_rows_of_several_groups(ctx, rows):
    l = normal(rows, 8200, "bf16", rows)
    l[rows - 1] = -torch.inf
    l[rows - 2, 1:] = -torch.inf
    check(ctx, l, 0.8, seed=1)
    check(ctx, l, 0.9, 40, 0.95, seed=2)                                # narrow sets
    check(ctx, l, [0.0 if r % 7 == 0 else 1.0 + r / 300 for r in range(rows)], 3000, 0.99, seed=3)   # wide ones
    check(ctx, l, 1.5, None, 0.9, 0.02, seed=4)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("V", [1 << 20, (1 << 20) - 9])
def test_longest_rows(ctx, t, V):
    l = normal(2, V, t, V)
    l[1, V - 1] = 14.0   # ahead of the others
    check(ctx, l, seed=1)
    check(ctx, l, 0.8, 50, 0.9, seed=2)
    check(ctx, l, 1.0, None, 0.9, seed=3)
    check(ctx, l, 1.0, 300000, 0.99, seed=4)
    check(ctx, l, 1.2, V - 1, seed=5, u=1.0)
    check(ctx, l, 1.0, None, 0.999, 1e-4, seed=6)
    check(ctx, torch.zeros_like(l), 1.0, 700000, 0.5, seed=7)
