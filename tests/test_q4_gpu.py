"""aq_q4_forward against its definition in 64 bits.

Tolerances, from the arithmetic.  Floating x: a group's sum is formed from
x (16 + q) and -(16 + zero) x in fp32, whose partial sums are up to about
24 / 4.6 = 5 times the result's; with some ten roundings of 2^-25 of those on
the way (random signs: times 3) and the scaled sums after them the error is
about 1e-6 of the result's norm; 2e-6 is asked.  8-bit whole numbers are
summed exactly, so only the scalings (two roundings) and the sum over the
groups remain: 5e-7.  The output's rounding adds 2^-11 (f16) or 2^-8 (bf16)
at most, 0.6 of that in the norm.  No value is further off than its terms
allow: 2^-18 of the sum of their magnitudes, 62 |x| scale each."""

import numpy as np
import pytest
import torch

import aqmi

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8,
         "e4m3": torch.float8_e4m3fn}
OUT = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def ctx():
    return aqmi.Context(0)


def matrix(N, K, G, zeros, bias, seed):
    r = np.random.default_rng(seed)
    groups = -(-K // G)
    codes = r.integers(0, 256, (N, (K + 1) // 2), dtype=np.uint8)
    scale = (r.uniform(0.5, 1.5, (N, groups)) / np.sqrt(K)).astype(np.float16)
    zero = r.integers(0, 16, (N, groups), dtype=np.uint8) if zeros else None
    b = r.standard_normal(N).astype(np.float32) if bias else None
    return codes, scale, zero, b


def dense(codes, scale, zero, K, G):
    q = np.stack((codes & 15, codes >> 4), 2).reshape(len(codes), -1)[:, :K].astype(np.float64)
    at = np.arange(K) // G
    z = 8 if zero is None else zero.astype(np.float64)[:, at]
    return (q - z) * scale.astype(np.float64)[:, at]


def rows(M, K, t, xg, seed, ld=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, ld or K, generator=g)
    s = None
    if t in ("i8", "e4m3"):
        most = 127 if t == "i8" else 448
        x = (x * most / 3.5).clamp(-most, most)
        x = x.round() if t == "i8" else x
        s = (torch.rand(M, -(-K // xg) if xg else 1, generator=g) + 0.5).cuda()
    return x.to(TYPES[t]).cuda()[:, :K], s


def check(ctx, N, K, G, M, t, out="f32", zeros=False, bias=False, xg=0, x_ld=None, y_ld=None):
    codes, scale, zero, b = matrix(N, K, G, zeros, bias, N + K)
    lin = aqmi.Q4Linear(ctx, codes, scale, K, G, zero, b)
    x, s = rows(M, K, t, xg, M, x_ld)
    full = torch.full((M, y_ld or N), 7.0, dtype=TYPES[out], device="cuda")
    y = full[:, :N]
    lin.forward(x, y, s, xg)
    torch.cuda.synchronize()
    xd = x.double().cpu().numpy()
    if s is not None:
        xd = xd * s.double().cpu().numpy()[:, np.arange(K) // (xg or K)]
    ref = xd @ dense(codes, scale, zero, K, G).T + (0 if b is None else b.astype(np.float64))
    got = y.double().cpu().numpy()
    rel = (5e-7 if t == "i8" else 2e-6) + 0.6 * OUT[out]
    assert np.linalg.norm(got - ref) <= rel * np.linalg.norm(ref)
    worst = 62 * np.abs(xd) @ np.repeat(scale.astype(np.float64), G, 1)[:, :K].T
    assert np.all(np.abs(got - ref) <= 2.0 ** -18 * worst + OUT[out] * np.abs(ref) + 1e-7 * np.abs(ref) + 2.0 ** -25)
    if y_ld:
        assert bool((full[:, N:] == 7).all())   # nothing is written past a row's end


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("N,K,M", [(1, 1, 1), (17, 33, 3), (64, 256, 16), (100, 1000, 5), (129, 999, 33), (33, 128, 70),
                                   (256, 2048, 64), (40, 2500, 1)])
def test_against_64_bits(ctx, t, G, zeros, N, K, M):
    check(ctx, N, K, G, M, t, zeros=zeros, bias=zeros)


@pytest.mark.parametrize("t", ["i8", "e4m3"])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("xg", [32, 64, 128])
def test_scales_of_8_bit_rows(ctx, t, G, xg):
    check(ctx, 80, 1000, G, 4, t, zeros=True, xg=xg)
    check(ctx, 48, 512, G, 40, t, xg=xg)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("out", OUT)
def test_types_and_strides(ctx, t, out):
    check(ctx, 77, 513, 64, 6, t, out, bias=True, x_ld=515, y_ld=79)
    check(ctx, 96, 640, 32, 50, t, out, zeros=True, x_ld=641, y_ld=101)
    check(ctx, 64, 384, 128, 20, t, out)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("N,M", [(8203, 1), (8203, 6), (16397, 5), (24601, 2)])
def test_long_matrices(ctx, t, G, N, M):
    """Sizes where a block takes one, two or four tiles of rows, the last one with fewer."""
    check(ctx, N, 1100, G, M, t, zeros=True)


@pytest.mark.parametrize("t", TYPES)
def test_long_matrices_and_many_rows(ctx, t):
    check(ctx, 16401, 300, 128, 70, t, bias=True)


def test_many_rows_of_x(ctx):
    check(ctx, 48, 256, 64, 1000, "bf16", "bf16")


def test_the_row_that_the_norm_writes(ctx):
    """A normalised row in 8 bits goes straight into the product."""
    M, K, N = 3, 1000, 50
    codes, scale, zero, b = matrix(N, K, 64, True, True, 5)
    lin = aqmi.Q4Linear(ctx, codes, scale, K, 64, zero, b)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    for dt in (torch.int8, torch.float8_e4m3fn):
        q, s = torch.empty((M, K), dtype=dt, device="cuda"), torch.empty((M, -(-K // 64)), device="cuda")
        y = torch.empty((M, N), device="cuda")
        aqmi.add_rmsnorm(ctx, x, None, 1e-6, q=q, scale=s, group=64)
        lin.forward(q, y, s, 64)
        xd = q.double().cpu().numpy() * s.double().cpu().numpy()[:, np.arange(K) // 64]
        ref = xd @ dense(codes, scale, zero, K, 64).T + b
        assert np.linalg.norm(y.double().cpu().numpy() - ref) <= 2e-6 * np.linalg.norm(ref)


def test_non_finite_rows_stay_alone(ctx):
    codes, scale, zero, b = matrix(40, 300, 64, False, False, 3)
    lin = aqmi.Q4Linear(ctx, codes, scale, 300, 64)
    for t in ("f32", "f16", "bf16"):
        x, _ = rows(20, 300, t, 0, 1)
        x = x.clone()
        y, z = (torch.empty((20, 40), device="cuda") for _ in range(2))
        lin.forward(x, y)
        x[3, 7], x[17, 299] = float("nan"), float("inf")
        lin.forward(x, z)
        keep = [i for i in range(20) if i not in (3, 17)]
        assert torch.equal(y[keep], z[keep]) and z[3].isnan().all() and z[17].isnan().all()


def test_quantize_round_trip():
    w = np.random.default_rng(0).standard_normal((9, 100)).astype(np.float32)
    for zeros in (False, True):
        codes, scale, zero = aqmi.q4_quantize(w, 32, zeros)
        step = np.repeat(scale.astype(np.float64), 32, 1)[:, :100]
        # half a step, and with zeros the zero's own rounding at the range's ends
        assert np.all(np.abs(dense(codes, scale, zero, 100, 32) - w) <= (1.01 if zeros else 0.51) * step)


def test_refusals(ctx):
    codes, scale, zero, b = matrix(32, 64, 32, True, True, 1)
    lib = ctx.lib
    import ctypes as C

    def upload(N=32, K=64, G=32, c=codes.ctypes.data, s=scale.ctypes.data, z=zero.ctypes.data):
        h = C.c_void_p()
        st = lib.aq_q4_upload(ctx.h, N, K, G, c, s, z, None, C.byref(h))
        if st == 0:
            lib.aq_q4_release(h)
        return st

    assert upload() == 0
    high = zero.copy()
    high[31, 1] = 16
    for bad, status in [(dict(c=None), 1), (dict(s=None), 1), (dict(G=16), 1), (dict(N=0), 2), (dict(K=0), 2),
                        (dict(N=(1 << 24) + 1), 2), (dict(N=1 << 24, K=1 << 11), 2), (dict(z=high.ctypes.data), 1)]:
        assert upload(**bad) == status, bad
        assert "aq_q4_upload" in lib.aq_last_error(ctx.h).decode()
    lin = aqmi.Q4Linear(ctx, codes, scale, 64, 32, zero, b)
    x, y = torch.zeros((4, 64), device="cuda"), torch.zeros((4, 32), device="cuda")
    q, s = torch.zeros((4, 64), dtype=torch.int8, device="cuda"), torch.zeros((4, 2), device="cuda")

    def forward(t=0, x=x.data_ptr(), ld=64, xs=None, xg=0, M=4, yt=0, y=y.data_ptr(), y_ld=32):
        return lib.aq_q4_forward(ctx.h, lin.h, t, x, ld, xs, xg, M, yt, y, y_ld)

    assert forward() == 0 and forward(M=0, x=None, y=None) == 0
    assert forward(t=3, x=q.data_ptr(), xs=s.data_ptr(), xg=32) == 0
    for bad, status in [(dict(t=5), 1), (dict(yt=3), 1), (dict(x=None), 1), (dict(y=None), 1), (dict(t=3), 1),
                        (dict(xs=s.data_ptr()), 1), (dict(t=3, xs=s.data_ptr(), xg=16), 1), (dict(ld=63), 2),
                        (dict(y_ld=31), 2), (dict(M=-1), 2), (dict(M=(1 << 20) + 1), 2)]:
        assert forward(**bad) == status, bad
        assert "aq_q4_forward" in lib.aq_last_error(ctx.h).decode()
    with pytest.raises(ValueError):
        lin.forward(q, y)
    with pytest.raises(ValueError):
        lin.forward(x[:, :63], y)
    with pytest.raises(ValueError):
        aqmi.Q4Linear(ctx, codes, scale, 66, 32)
