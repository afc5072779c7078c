"""aq_i8_forward against its definition in 64 bits.

Tolerances, from the arithmetic.  The sums are whole numbers and exact; their
conversion to fp32, the scalings with either scale and the bias's addition
round once each: 4 * 2^-24 of the product's magnitude (and of the result where
the bias is added), 2.5e-7; 3e-7 is asked of every value.  A floating row's
scale is rounded once more: 2^-24, within the same.  The output's rounding adds
2^-11 (f16) or 2^-8 (bf16) of the value, and below the least normal f16 half a
step of 2^-24."""

import ctypes as C

import numpy as np
import pytest
import torch

import aqmi

pytestmark = pytest.mark.gpu

TYPES = {"i8": torch.int8, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
OUT = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def ctx():
    return aqmi.Context(0)


def matrix(N, K, bias, seed):
    r = np.random.default_rng(seed)
    w = r.integers(-128, 128, (N, K), dtype=np.int8)
    scale = (r.uniform(0.5, 1.5, N) / 64 / np.sqrt(K)).astype(np.float32)
    return w, scale, r.standard_normal(N).astype(np.float32) if bias else None


def rows(M, K, t, seed, ld=None):
    g = torch.Generator().manual_seed(seed)
    if t == "i8":
        x = torch.randint(-128, 128, (M, ld or K), generator=g, dtype=torch.int8)
        return x.cuda()[:, :K], (torch.rand(M, generator=g) + 0.5).cuda() / 64
    x = torch.randn(M, ld or K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))
    return x.to(TYPES[t]).cuda()[:, :K], None


def eight(x):
    """The 8-bit rows and scales of floating ones, in exact arithmetic: 254 |x| against (2 q + 1) max, both whole
    multiples of one power of two below 2^53."""
    x = x.double().cpu().numpy()
    most = np.abs(x).max(1, keepdims=True)
    safe = np.where(most > 0, most, 1)
    q = np.floor(np.abs(x) * 127 / safe)
    for _ in range(2):   # the floor, corrected where the quotient was rounded over it
        q = np.where(127 * np.abs(x) < q * safe, q - 1, np.where(127 * np.abs(x) >= (q + 1) * safe, q + 1, q))
    left = 254 * np.abs(x) - 2 * q * safe
    q = q + ((left > safe) | ((left == safe) & (q % 2 == 1)))
    return np.where(most > 0, np.copysign(q, x), 0), most[:, 0] / 127


def reference(w, scale, bias, x, s):
    q, per = (x.cpu().numpy().astype(np.float64), s.double().cpu().numpy()) if s is not None else eight(x)
    y = (q @ w.astype(np.float64).T) * per[:, None] * scale.astype(np.float64)
    return y, y if bias is None else y + bias


def check(ctx, N, K, M, t, out="f32", bias=False, x_ld=None, y_ld=None):
    w, scale, b = matrix(N, K, bias, N + K)
    lin = aqmi.I8Linear(ctx, w, scale, b)
    x, s = rows(M, K, t, M, x_ld)
    full = torch.full((M, y_ld or N), 7.0, dtype=TYPES[out], device="cuda")
    lin.forward(x, full[:, :N], s)
    torch.cuda.synchronize()
    product, ref = reference(w, scale, b, x, s)
    got = full[:, :N].double().cpu().numpy()
    allowed = 3e-7 * (np.abs(product) + np.abs(ref)) + OUT[out] * np.abs(ref) + (2.0 ** -25 if out == "f16" else 0)
    assert np.all(np.abs(got - ref) <= allowed)
    if y_ld:
        assert bool((full[:, N:] == 7).all())   # nothing is written past a row's end


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("N,K,M", [(1, 1, 1), (17, 33, 3), (64, 256, 16), (100, 1000, 5), (129, 999, 33), (33, 128, 70),
                                   (256, 2048, 64), (40, 2500, 1), (1000, 1001, 17), (300, 640, 300), (513, 192, 257)])
def test_against_64_bits(ctx, t, bias, N, K, M):
    check(ctx, N, K, M, t, bias=bias)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("out", OUT)
@pytest.mark.parametrize("M", [6, 50, 140, 600])
def test_types_and_strides(ctx, t, out, M):
    check(ctx, 77, 513, M, t, out, bias=True, x_ld=515, y_ld=79)
    check(ctx, 96, 640, M, t, out, x_ld=656, y_ld=101)
    check(ctx, 64, 384, M, t, out)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("N,K,M", [(8203, 1100, 1), (16397, 320, 5), (8208, 300, 70), (2050, 4100, 130), (1030, 1024, 1030)])
def test_long_matrices(ctx, t, N, K, M):
    check(ctx, N, K, M, t, bias=True)


@pytest.mark.parametrize("M", [1, 16, 17, 64, 65, 300])
def test_the_longest_sums_fit(ctx, M):
    """2^17 - 1 products of -128 and -128, just below 2^31."""
    K = (1 << 17) - 1
    lin = aqmi.I8Linear(ctx, np.full((3, K), -128, np.int8), np.ones(3, np.float32))
    x, s, y = torch.full((M, K), -128, dtype=torch.int8, device="cuda"), torch.ones(M, device="cuda"), torch.zeros((M, 3), device="cuda")
    lin.forward(x, y, s)
    assert bool((y == float(np.float32(128 * 128 * K))).all())
    with pytest.raises(aqmi.AqError):
        aqmi.I8Linear(ctx, np.zeros((1, K + 1), np.int8), np.ones(1, np.float32))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_values_half_way_between_whole_numbers(ctx, t):
    """Rows of max 254 * 2^e: x = (2 n + 1) 2^e is half way between two codes and goes to the even one; in f32 its
    neighbours go to theirs.  Read back through the unit matrix."""
    n = np.arange(-127, 127)
    K = 1 + 3 * len(n)
    w = np.eye(K, dtype=np.int8)
    lin = aqmi.I8Linear(ctx, w, np.ones(K, np.float32))
    x = np.zeros((5, K), np.float32)
    for i, e in enumerate((0, -3, 5, -100 if t != "f16" else -8, 90 if t != "f16" else 7)):
        half = ((2 * n + 1) * 2.0 ** e).astype(np.float32)
        x[i] = np.concatenate(([254 * 2.0 ** e], half, *((np.nextafter(half, np.float32(d)) if t == "f32" else half) for d in (np.inf, -np.inf))))
    xt = torch.from_numpy(x).to(TYPES[t]).cuda()
    y = torch.empty((5, K), device="cuda")
    lin.forward(xt, y)
    q, per = eight(xt)
    assert np.array_equal(np.rint(y.double().cpu().numpy() / per[:, None]), q)


@pytest.mark.parametrize("M", [3, 40])
def test_rows_of_zeros_and_of_values_that_are_not_finite(ctx, M):
    w, scale, b = matrix(40, 300, True, 3)
    lin = aqmi.I8Linear(ctx, w, scale, b)
    for t in ("f32", "f16", "bf16"):
        x, _ = rows(M, 300, t, 1)
        x = x.clone()
        y, z = (torch.empty((M, 40), device="cuda") for _ in range(2))
        lin.forward(x, y)
        x[0] = 0
        x[1, 7], x[2, 299] = float("nan"), float("-inf")
        lin.forward(x, z)
        assert torch.equal(y[3:], z[3:]) and z[1].isnan().all() and z[2].isnan().all()
        assert torch.equal(z[0].cpu(), torch.from_numpy(b))


def test_smallest_and_largest_rows(ctx):
    """Rows whose largest value is subnormal, or next to fp32's end."""
    w, scale, _ = matrix(33, 70, False, 9)
    lin = aqmi.I8Linear(ctx, w, scale)
    x, _ = rows(4, 70, "f32", 2)
    x = x / x.abs().amax(1, keepdim=True) * torch.tensor([[2.0 ** -149], [2.0 ** -130], [3.4e38], [1e-30]], device="cuda")
    y = torch.empty((4, 33), device="cuda")
    lin.forward(x, y)
    q, per = eight(x)
    per = per.astype(np.float32).astype(np.float64)   # a scale below the least normal value keeps fewer bits
    ref = (q @ w.astype(np.float64).T) * per[:, None] * scale.astype(np.float64)
    # the scales' product, and the result, round to multiples of 2^-149
    sums = np.abs(q @ w.astype(np.float64).T)
    got = y.double().cpu().numpy()
    # A result beyond fp32's range by more than the tolerance has no finite value: it is an infinity.  (The row next to
    # the end has sums over 127, so its largest results are up to some 1.1 times that row's 3.4e38.)
    beyond = np.abs(ref) * (1 - 3e-7) >= 2.0 ** 128
    assert np.array_equal(got[beyond], np.copysign(np.inf, ref[beyond])) and not beyond[[0, 1, 3]].any()
    assert np.all(np.abs(got - ref)[~beyond] <= (3e-7 * np.abs(ref) + 2.0 ** -150 * (sums + 1))[~beyond])


def test_the_row_that_the_norm_writes(ctx):
    """A normalised row in 8 bits with one scale goes straight into the product."""
    M, K, N = 3, 1000, 50
    w, scale, b = matrix(N, K, True, 5)
    lin = aqmi.I8Linear(ctx, w, scale, b)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    q, s, y = torch.empty((M, K), dtype=torch.int8, device="cuda"), torch.empty((M, 1), device="cuda"), torch.empty((M, N), device="cuda")
    aqmi.add_rmsnorm(ctx, x, None, 1e-6, q=q, scale=s)
    lin.forward(q, y, s)
    product, ref = reference(w, scale, b, q, s[:, 0])
    assert np.all(np.abs(y.double().cpu().numpy() - ref) <= 3e-7 * (np.abs(product) + np.abs(ref)))


def test_quantize_round_trip(ctx):
    w = np.random.default_rng(0).standard_normal((9, 100)).astype(np.float32)
    w[4] = 0
    codes, scale = aqmi.i8_quantize(w)
    assert np.all(np.abs(codes * scale.astype(np.float64)[:, None] - w) <= 0.5001 * scale[:, None])
    assert np.abs(codes).max() == 127 and not codes[4].any()


def test_refusals(ctx):
    w, scale, b = matrix(32, 64, True, 1)
    lib = ctx.lib

    def upload(N=32, K=64, c=w.ctypes.data, s=scale.ctypes.data):
        h = C.c_void_p()
        st = lib.aq_i8_upload(ctx.h, N, K, c, s, None, C.byref(h))
        if st == 0:
            lib.aq_i8_release(h)
        return st

    assert upload() == 0
    for bad, status in [(dict(c=None), 1), (dict(s=None), 1), (dict(N=0), 2), (dict(K=0), 2), (dict(K=1 << 17), 2),
                        (dict(N=(1 << 24) + 1), 2), (dict(N=1 << 24, K=1 << 11), 2)]:
        assert upload(**bad) == status, bad
        assert "aq_i8_upload" in lib.aq_last_error(ctx.h).decode()
    lin = aqmi.I8Linear(ctx, w, scale, b)
    x, y = torch.zeros((4, 64), device="cuda"), torch.zeros((4, 32), device="cuda")
    q, s = torch.zeros((4, 64), dtype=torch.int8, device="cuda"), torch.zeros(4, device="cuda")

    def forward(t=0, x=x.data_ptr(), ld=64, xs=None, M=4, yt=0, y=y.data_ptr(), y_ld=32):
        return lib.aq_i8_forward(ctx.h, lin.h, t, x, ld, xs, M, yt, y, y_ld)

    assert forward() == 0 and forward(M=0, x=None, y=None) == 0
    assert forward(t=3, x=q.data_ptr(), xs=s.data_ptr()) == 0
    for bad, status in [(dict(t=4), 1), (dict(t=5), 1), (dict(yt=3), 1), (dict(x=None), 1), (dict(y=None), 1), (dict(t=3), 1),
                        (dict(xs=s.data_ptr()), 1), (dict(ld=63), 2), (dict(y_ld=31), 2), (dict(M=-1), 2),
                        (dict(M=(1 << 20) + 1), 2)]:
        assert forward(**bad) == status, bad
        assert "aq_i8_forward" in lib.aq_last_error(ctx.h).decode()
    for bad in (lambda: lin.forward(q, y), lambda: lin.forward(x, y, s), lambda: lin.forward(x[:, :63], y),
                lambda: lin.forward(q, y, s[:3]), lambda: aqmi.I8Linear(ctx, w, scale[:3]),
                lambda: aqmi.I8Linear(ctx, w, scale, b[:3]), lambda: aqmi.I8Linear(ctx, w.astype(np.float32), scale)):
        with pytest.raises(ValueError):
            bad()
