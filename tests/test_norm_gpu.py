"""aq_add_rmsnorm against its definition in 64 bits.

Tolerances, from the arithmetic: h is one fp32 addition rounded to the type,
so it equals the reference's.  y takes a sum of squares in fp32 (each thread
at most 32 fused additions and then a tree: relative error of the sum below
(32 + 12) * 2^-24, half of that in its root, below 1.4e-6 with the roundings
of the mean, the root and the division), two products and the rounding to the
type: 2^-24 (f32), 2^-11 (f16), 2^-8 (bf16) of |y|.  A scale has the same
bound of 1.6e-6.  q is the nearest 8-bit value of p * (L / max |p|), three
roundings of 2^-24 away from the exact quotient: at most 127 * 3 * 2^-24 =
2.3e-5 of a step for I8; e4m3's steps are at least 2^-4 of the value, so
2.9e-6 of a step.  So q is held to 0.5 + 1e-4 steps of its exact quotient."""

import numpy as np
import pytest
import torch

import aqmi

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
REL = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
EIGHT = {"i8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


@pytest.fixture(scope="module")
def ctx():
    return aqmi.Context(0)


def make(M, D, t, seed, ld=None):
    g = torch.Generator().manual_seed(seed)
    ld = ld or D
    full = [torch.randn(M, ld, generator=g).to(TYPES[t]).cuda() for _ in range(2)]
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(TYPES[t]).cuda()
    return full[0][:, :D], full[1][:, :D], w


def check(ctx, x, r, w, t, kind, group, eps=1e-6, sum=None, y=None):
    M, D = x.shape
    xs, rs = x.clone(), None if r is None else r.clone()
    sum = torch.full((M, D), 7, dtype=x.dtype, device="cuda") if sum is None else sum
    y = torch.full((M, D), 7, dtype=x.dtype, device="cuda") if y is None else y
    dt, most = EIGHT[kind]
    groups = -(-D // group) if group else 1
    q = torch.empty((M, D), dtype=dt, device="cuda")
    scale = torch.empty((M, groups), device="cuda")
    aqmi.add_rmsnorm(ctx, x, w, eps, residual=r, sum=sum, y=y, q=q, scale=scale, group=group)
    torch.cuda.synchronize()

    h = (xs.float() + rs.float()).to(x.dtype) if rs is not None else xs
    assert torch.equal(sum, h)
    h = h.double().cpu().numpy()
    p = h * (1 if w is None else w.double().cpu().numpy())
    ref = p / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    got = y.double().cpu().numpy()
    tiny = 2.0 ** -25 if t == "f16" else 0.0   # half a step of f16's subnormals
    assert np.all(np.abs(got - ref) <= (1.6e-6 + REL[t]) * np.abs(ref) + tiny)
    starts = np.arange(0, D, group or D)
    per = np.maximum.reduceat(np.abs(ref), starts, axis=1) / most
    s = scale.double().cpu().numpy()
    assert np.all(np.abs(s - per) <= 1.6e-6 * per)
    wide = np.repeat(per, np.diff(np.append(starts, D)), axis=1)
    exact = np.divide(ref, wide, out=np.zeros_like(ref), where=wide > 0)
    step = 1.0 if kind == "i8" else np.exp2(np.maximum(np.frexp(exact)[1] - 1, -6) - 3.0)
    assert np.all(np.abs(q.double().cpu().numpy() - exact) <= (0.5 + 1e-4) * step)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kind,group", [("i8", 32), ("i8", 0), ("e4m3", 64), ("e4m3", 128), ("e4m3", 0), ("i8", 128)])
@pytest.mark.parametrize("M,D", [(1, 1), (3, 7), (5, 33), (1, 512), (7, 1001), (4, 1024), (2, 1999), (9, 4096),
                                 (3, 8191), (2, 16384), (1, 30000), (2, 40001)])
def test_against_64_bits(ctx, t, kind, group, M, D):
    x, r, w = make(M, D, t, D + M)
    check(ctx, x, r, w, t, kind, group)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [1000, 3000, 8000])
def test_batches_of_rows(ctx, t, D):
    """More rows than the few that get a wider block each."""
    x, r, w = make(515, D, t, D)
    check(ctx, x, r, w, t, "i8", 32)
    check(ctx, x, None, w, t, "e4m3", 0)


def test_more_rows_than_a_grid_takes(ctx):
    """Two launches; the last rows against the same rows alone."""
    M, D = (1 << 21) + 5, 40
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn((M, D), generator=g, device="cuda").bfloat16()
    r = torch.randn((M, D), generator=g, device="cuda").bfloat16()
    w = (1 + 0.3 * torch.randn(D, generator=g, device="cuda")).bfloat16()

    def run(x, r):
        y, q = torch.empty_like(x), torch.empty(x.shape, dtype=torch.int8, device="cuda")
        h, scale = torch.empty_like(x), torch.empty((len(x), 2), device="cuda")
        aqmi.add_rmsnorm(ctx, x, w, 1e-6, residual=r, sum=h, y=y, q=q, scale=scale, group=32)
        return h, y, q, scale

    for whole, part in zip(run(x, r), run(x[-9:], r[-9:])):
        assert torch.equal(whole[-9:], part)
    for whole, part in zip(run(x, r), run(x[:7], r[:7])):
        assert torch.equal(whole[:7], part)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D,ld", [(100, 103), (1024, 1025), (2050, 2064), (40000, 40003)])
def test_strided_rows_in_place(ctx, t, D, ld):
    """x read at odd offsets; h written over x, y over the residual."""
    x, r, w = make(6, D, t, D, ld)
    check(ctx, x, r, w, t, "i8", 64, sum=x, y=r)
    x, r, w = make(6, D, t, D + 1, ld)
    check(ctx, x, None, None, t, "e4m3", 32)
    x, r, w = make(6, D, t, D + 2, ld)
    check(ctx, x, r, w, t, "e4m3", 0, sum=r)


@pytest.mark.parametrize("D", [48, 300, 3001, 33000])
def test_zero_and_non_finite_rows(ctx, D):
    x, _, w = make(5, D, "f32", 3)
    x = x.clone()
    x[0] = 0
    x[1, D // 2] = float("nan")
    x[2, D - 1] = float("inf")
    x[3, :32] = 0
    y, scale = torch.empty_like(x), torch.empty((5, -(-D // 32)), device="cuda")
    for dt in (torch.int8, torch.float8_e4m3fn):
        q = torch.empty((5, D), dtype=dt, device="cuda")
        aqmi.add_rmsnorm(ctx, x, w, 1e-6, y=y, q=q, scale=scale, group=32)
        assert not y[0].any() and not q[0].float().any() and not scale[0].any()
        assert y[1].isnan().all() and scale[1].isnan().all()
        assert y[2, D - 1].isnan() and not y[2, :D - 1].any()
        assert scale[2, -1].isnan() and not scale[2, :-1].any()
        assert scale[3, 0] == 0 and not q[3, :32].float().any() and y[3, 32:].isfinite().all() and scale[3, 1] > 0
    w[5] = float("nan")
    aqmi.add_rmsnorm(ctx, x, w, 1e-6, y=y, q=q, scale=scale, group=32)
    assert scale[4, 0].isnan() and scale[4, 1:].isfinite().all() and y[4, 5].isnan()


def test_sum_alone_and_empty_batch(ctx):
    x, r, _ = make(3, 77, "bf16", 1)
    h = torch.empty_like(x)
    aqmi.add_rmsnorm(ctx, x, None, 0.0, residual=r, sum=h)
    assert torch.equal(h, x + r)
    e = torch.empty((0, 77), dtype=torch.bfloat16, device="cuda")
    aqmi.add_rmsnorm(ctx, e, None, 1e-6, y=e)


def test_another_stream(ctx):
    x, r, w = make(64, 2048, "bf16", 9)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        check(ctx, x, r, w, "bf16", "i8", 32)


def test_refusals(ctx):
    x, r, w = make(4, 64, "f32", 2)
    q, s = torch.empty((4, 64), dtype=torch.int8, device="cuda"), torch.empty((4, 2), device="cuda")
    lib, p = ctx.lib, x.data_ptr()

    def call(type=0, x=p, x_ld=64, res=None, res_ld=64, M=4, D=64, eps=1e-6, sum=None, sum_ld=64, y=None, y_ld=64,
             q_type=3, group=32, q=q.data_ptr(), scale=s.data_ptr()):
        return lib.aq_add_rmsnorm(ctx.h, type, x, x_ld, res, res_ld, None, M, D, eps, sum, sum_ld, y, y_ld, q_type,
                                  group, q, scale)

    assert call() == 0
    other = r.data_ptr()
    for bad, status in [(dict(type=3), 1), (dict(type=9), 1), (dict(x=None), 1), (dict(scale=None), 1),
                        (dict(q=None), 1), (dict(q=None, scale=None), 1), (dict(q_type=2), 1), (dict(group=16), 1),
                        (dict(group=-1), 1), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1), (dict(M=-1), 2),
                        (dict(D=0), 2), (dict(D=(1 << 30) + 1), 2), (dict(x_ld=63), 2), (dict(res=other, res_ld=63), 2),
                        (dict(y=other, y_ld=63), 2), (dict(sum=other, y=other), 1), (dict(sum=p, sum_ld=65), 2),
                        (dict(y=p, y_ld=65), 2), (dict(res=other, y=other, y_ld=65), 2)]:
        assert call(**bad) == status, bad
        assert "aq_add_rmsnorm" in lib.aq_last_error(ctx.h).decode()
    assert lib.aq_add_rmsnorm(None, 0, p, 64, None, 0, None, 4, 64, 1e-6, None, 0, p, 64, 3, 0, None, None) == 1
    with pytest.raises(ValueError):
        aqmi.add_rmsnorm(ctx, x, w[:3], 1e-6, y=x)
    with pytest.raises(ValueError):
        aqmi.add_rmsnorm(ctx, x, w, 1e-6, q=q, scale=s, group=64)
    with pytest.raises(TypeError):
        aqmi.add_rmsnorm(ctx, x, w, 1e-6, y=x.half())
