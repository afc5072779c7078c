"""aq_i8_forward at the ends of fp32's range, against its definition in 64 bits.

The sum's conversion to fp32, the scalings with either scale, a floating row's
own scale and the bias's addition round once each: 5 * 2^-24 of the product's
magnitude and of the result, below 3e-7; below the least normal value a result
rounds to a multiple of 2^-149.  A result beyond fp32's range is an infinity."""

import numpy as np
import pytest
import torch

import aqmi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return aqmi.Context(0)


def near(got, ref, product):
    got = got.double().cpu().numpy()
    beyond = np.abs(ref) * (1 - 3e-7) >= 2.0 ** 128
    assert np.array_equal(got[beyond], np.copysign(np.inf, ref[beyond]))
    assert np.all(np.abs(got - ref)[~beyond] <= (3e-7 * (np.abs(ref) + np.abs(product)) + 2.0 ** -149)[~beyond])
    return beyond


FAR = np.array([3e38, 1e30, 2.0 ** 97, 2.0 ** 96, 1.0, 1e-30, 2.0 ** -130, 2.0 ** -149], np.float32)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("N,K,M", [(19, 100, 9), (40, 131, 50), (70, 1000, 140), (270, 208, 270), (50, 2100, 90)])
def test_scales_far_from_one(ctx, bias, N, K, M):
    """One scale that the other makes up for: the product has a finite value, whichever of the two is the large one."""
    r = np.random.default_rng(M)
    w = r.integers(-128, 128, (N, K), dtype=np.int8)
    scale = np.resize(FAR, N) * r.choice([1, -1], N).astype(np.float32)
    b = r.standard_normal(N).astype(np.float32) if bias else None
    lin = aqmi.I8Linear(ctx, w, scale, b)
    g = torch.Generator().manual_seed(M)
    x = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8)
    xs = torch.from_numpy(np.resize(np.roll(FAR, 3)[[0, 5, 2, 7, 1, 6, 3, 4, 0]], M).astype(np.float32))
    y = torch.empty((M, N), device="cuda")
    lin.forward(x.cuda(), y, xs.cuda())
    ref = (x.numpy().astype(np.float64) @ w.astype(np.float64).T) * xs.double().numpy()[:, None] * scale.astype(np.float64)
    beyond = near(y, ref if b is None else ref + b, ref)
    assert beyond.any() and not beyond.all()


@pytest.mark.parametrize("M", [1, 30, 200])
def test_small_rows_with_large_weights(ctx, M):
    """Floating rows of some 1e-33 with weights of some 1e33."""
    r = np.random.default_rng(M)
    w = r.standard_normal((33, 70)).astype(np.float32) * np.float32(1e33)
    codes, scale = aqmi.i8_quantize(w)
    lin = aqmi.I8Linear(ctx, codes, scale)
    x = torch.randn((M, 70), generator=torch.Generator().manual_seed(M)) * 1e-33
    y = torch.empty((M, 33), device="cuda")
    lin.forward(x.cuda(), y)
    xd = x.double().numpy()
    most = np.abs(xd).max(1, keepdims=True)
    q = np.rint(xd * 127 / most)   # (no value of these is half way between two codes)
    assert np.abs(np.abs(xd * 127 / most - np.floor(xd * 127 / most)) - 0.5).min() > 1e-9
    ref = (q @ codes.astype(np.float64).T) * (most / 127) * scale.astype(np.float64)
    near(y, ref, ref)


@pytest.mark.parametrize("t", ["i8", "bf16"])
@pytest.mark.parametrize("M", [16, 40, 140])
def test_rows_farther_apart_than_32_bits(ctx, t, M):
    """The last rows of x and of y start past 2^32 bytes and 2^32 elements; the results are those of rows next to each other."""
    step, K, N = -(-(1 << 32) // (M - 1) // 16) * 16 + 16, 208, 270
    r = np.random.default_rng(M)
    lin = aqmi.I8Linear(ctx, r.integers(-128, 128, (N, K), dtype=np.int8), np.full(N, 1e-3, np.float32))
    g = torch.Generator().manual_seed(M)
    x, s = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8).cuda(), torch.rand(M, generator=g).cuda()
    if t != "i8":
        x, s = x.bfloat16(), None
    near_y = torch.empty((M, N), dtype=torch.bfloat16, device="cuda")
    lin.forward(x, near_y, s)
    far_x = torch.empty(M * step, dtype=x.dtype, device="cuda").view(M, step)[:, :K]
    far_x.copy_(x)
    far_y = torch.empty(M * step, dtype=torch.bfloat16, device="cuda").view(M, step)[:, :N]
    lin.forward(far_x, far_y, s)
    assert torch.equal(far_y, near_y)


def test_results_past_32_bits(ctx):
    """600000 rows of 4096 columns: 2.4 G results, of large blocks."""
    M, K, N = 600000, 64, 4096
    r = np.random.default_rng(1)
    lin = aqmi.I8Linear(ctx, r.integers(-128, 128, (N, K), dtype=np.int8), np.full(N, 1e-3, np.float32))
    x = torch.randint(-128, 128, (1000, K), generator=torch.Generator().manual_seed(1), dtype=torch.int8).cuda().repeat(M // 1000, 1)
    s = torch.full((M,), 0.5, device="cuda")
    y = torch.empty((M, N), dtype=torch.bfloat16, device="cuda")
    lin.forward(x, y, s)
    want = torch.empty((1000, N), dtype=torch.bfloat16, device="cuda")
    lin.forward(x[:1000], want, s[:1000])
    assert bool((y.view(-1, 1000, N) == want).all())
