"""aq_sample against its definition.

Two references.  One takes the fp32 weights e = 2^z as the device's exp2
gives them and does the rest in whole numbers with a sort: token for token
equal, no tolerance, since every sum is of whole numbers.  The other is the
definition in 64 bits throughout: an fp32 z has three roundings (difference,
log2(e) / T, product) of 2^-24 of at most |z| < 32 and the exp2 one of 2^-23,
so a weight is off by at most 32 * 3 * 2^-24 * ln 2 + 2^-23 < 4.2e-6 of
itself, plus 2^-31 of the largest for its rounding down; a running sum is off
by no more, 4.2e-6 + V * 2^-31 of the total.  The drawn token's interval of
the running weight must hold u within 2e-5 of the total (V <= 5000, both ends
and the total moved), and logp is off by at most 1.5e-5 + 2^-22 |logp|."""

import numpy as np
import pytest
import torch

import aqmi

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ctx():
    return aqmi.Context(0)


def weights32(l, t):
    """(z, e) in fp32 on the device, as numpy."""
    l = l.float()
    l = torch.where(l.isnan(), -torch.inf, l)
    top = l.amax(1, keepdim=True)
    per = torch.full_like(top, 1.4426950408889634) / torch.where(t > 0, t, 1.0)[:, None]
    z = torch.where(l == top, 0.0, l - top) * per
    return l.cpu().numpy(), z.cpu().numpy(), torch.where(l > -torch.inf, torch.exp2(z), 0.0).cpu().numpy()


def kept_weights(l, e, greedy, k, p, mp):
    """The whole-number weights of one row that the filters keep."""
    w = (e.astype(np.float64) * 2.0 ** 31).astype(np.int64)
    order = np.argsort(-l.astype(np.float64), kind="stable")
    order = order[w[order] > 0]
    if greedy:
        order = order[:1]
    elif 0 < k < len(l):
        order = order[:k]
    if p < 1:
        need = int(np.float32(p) * 2 ** 24) * int(w[order].sum()) >> 24 if p > 0 else 0
        before = np.cumsum(w[order]) - w[order]
        order = order[:max(1, int((before < need).sum()))]
    out = np.zeros_like(w)
    out[order] = w[order]
    if mp > 0:
        out[e < np.float32(min(mp, 1))] = 0
    return out


def check(ctx, logits, t=None, k=None, p=None, mp=None, seed=0, u=None):
    rows, V = logits.shape
    g = torch.Generator().manual_seed(seed)
    dev = lambda v, dt=torch.float32: None if v is None else torch.as_tensor(v, dtype=dt).expand(rows).contiguous().cuda()
    u = torch.rand(rows, generator=g).cuda() if u is None else dev(u)
    td, kd, pd, md = dev(t), dev(k, torch.int32), dev(p), dev(mp)
    token = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    logp = torch.full((rows,), 7.0, device="cuda")
    aqmi.sample(ctx, logits, u, token, td, kd, pd, md, logp)
    alone = torch.empty_like(token)
    aqmi.sample(ctx, logits, u, alone, td, kd, pd, md)
    torch.cuda.synchronize()
    assert torch.equal(token, alone)
    l, z, e = weights32(logits, torch.ones(rows, device="cuda") if td is None else td)
    one = lambda v, r, off: off if v is None else v[r].item()
    for r in range(rows):
        if not np.any(l[r] > -np.inf):
            assert token[r] == -1 and logp[r] == -np.inf
            continue
        w = kept_weights(l[r], e[r], not one(td, r, 1.0) > 0, one(kd, r, 0), one(pd, r, 1.0), one(md, r, 0.0))
        reach = np.cumsum(w)
        part = int(np.float32(min(max(u[r].item(), 0.0), 1 - 2.0 ** -24)) * 2 ** 24)
        want = int(np.searchsorted(reach, part * int(reach[-1]) >> 24, side="right"))
        assert token[r].item() == want, (r, token[r].item(), want)
        ref = z[r, want].astype(np.float64) * np.log(2) - np.log(reach[-1] / 2.0 ** 31)
        assert abs(logp[r].item() - ref) <= 2.0 ** -21 * max(1.0, abs(z[r, want]))
    return token, logp


def normal(rows, V, t, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(rows, V, generator=g)).to(TYPES[t]).cuda()


SIZES = [(1, 1), (3, 2), (2, 63), (5, 64), (4, 65), (7, 1000), (33, 1024), (2, 2049), (6, 4096), (3, 8192), (2, 16385),
         (1, 40000), (2, 70001)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,V", SIZES)
def test_filters(ctx, t, rows, V):
    l = normal(rows, V, t, V)
    check(ctx, l, seed=1)
    check(ctx, l, 0.7, seed=2)
    for k in (1, 2, 50, 5000):
        check(ctx, l, 0.8, k, seed=k)
    for p in (0.0, 1e-6, 0.3, 0.9, 0.999, 1 - 2.0 ** -24, 1.0):
        check(ctx, l, 1.3, None, p, seed=3)
    for mp in (0.01, 0.3, 1.0, 7.0):
        check(ctx, l, None, None, None, mp, seed=4)
    check(ctx, l, 0.9, 40, 0.95, 0.02, seed=5)
    check(ctx, l, 1.0, 400, 0.8, seed=6)


@pytest.mark.parametrize("V", [65, 1024, 3000, 9001, 20000, 70000, 300000])
@pytest.mark.parametrize("spread", [0.0, 0.05, 30.0])
def test_flat_and_peaked_rows(ctx, V, spread):
    """All equal (every tie goes by the index), nearly so, and one far ahead."""
    l = normal(3, V, "f32", V, spread)
    check(ctx, l, seed=1)
    check(ctx, l, 1.0, 50, seed=2)
    check(ctx, l, 1.0, V // 2, 0.5, seed=3)
    check(ctx, l, 2.0, None, 0.37, seed=4)
    check(ctx, l.bfloat16(), 0.5, 700, 0.9, 0.1, seed=5)


@pytest.mark.parametrize("V", [5000, 9001, 70000])
@pytest.mark.parametrize("ahead", [9.0, 14.0, 20.0])
def test_ends_in_a_far_tail(ctx, V, ahead):
    """One logit so far ahead that the kept set ends many bits below it."""
    l = normal(4, V, "f32", V, 1.5)
    l[:, V // 3] = ahead
    for p in (0.5, 0.97, 0.9999, 1 - 2.0 ** -24):
        check(ctx, l, 1.0, None, p, seed=1)
    check(ctx, l, 1.4, V // 3, 0.999, seed=2)
    check(ctx, l, 1.0, V // 2, None, 2.0 ** -22, seed=3)
    check(ctx, l, 1.2, V - 3, 0.999, 1e-5, seed=4)
    check(ctx, l, 1.0, V - 1, seed=5, u=1.0)


@pytest.mark.parametrize("V", [700, 9000, 40000])
def test_weights_at_the_edges_of_quarter_bits(ctx, V):
    """z in whole quarters down to below the last weight: a temperature of
    log2(e) makes z the logits' own difference."""
    l = -0.25 * (torch.arange(V) * 37 % 133).float().repeat(3, 1)
    l[1] *= 0.5
    l[2, : V // 2] = -31.0
    l[2, V // 2 :] = -31.000002
    l[2, V // 5] = 0.0
    l = l.cuda()
    t = 1.44269504
    some = int((l[0] >= -31).sum())
    check(ctx, l, t, seed=1)
    for k in (some - 1, some, some + 1, V - 1):
        check(ctx, l, t, k, seed=k, u=0.9999999)
    for p in (0.5, 0.999999, 1 - 2.0 ** -24):
        check(ctx, l, t, None, p, seed=2)
        check(ctx, l, t, V // 2, p, 2.0 ** -30, seed=3)


@pytest.mark.parametrize("V", [100, 2000, 6000, 33000, 70000])
def test_masks(ctx, V):
    lowest = torch.finfo(torch.float32).min
    l = normal(8, V, "f32", V)
    l[0] = -torch.inf                       # empty
    l[1] = float("nan")                     # nothing but NaN
    l[2, : V - 1] = -torch.inf              # the last alone
    l[3, V // 3:] = lowest                  # masked with the type's lowest
    l[4] = lowest                           # all at it: a flat row
    l[5, ::2] = -torch.inf
    l[5, 1::4] = float("nan")
    l[6, V // 2] = l[6, V - 1] = torch.inf  # two share the row
    l[7, 0] = torch.finfo(torch.float32).max
    for seed in range(3):
        token, _ = check(ctx, l, seed=seed)
        assert token[2] == V - 1 and token[3] < V // 3 and token[6] in (V // 2, V - 1) and token[7] == 0
        check(ctx, l, 0.7, 30, 0.8, 0.01, seed=seed)
        check(ctx, l, 1.1, None, 0.5, seed=seed)
        check(ctx, l, 0.0, seed=seed)


def test_rows_with_parameters_of_their_own(ctx):
    l = normal(9, 1500, "f16", 3)
    check(ctx, l, [0.5, 1.0, 0.0, -1.0, float("nan"), 2.0, 1e-30, 0.7, 1e6], [0, 1, -5, 50, 3, 1500, 2000, 10, 900],
          [0.9, 0.1, 1.0, 2.0, float("nan"), -1.0, 0.5, 0.0, 0.99], [0.0, -1.0, float("nan"), 0.2, 2.0, 0.0, 0.1, 0.5, 1e-9])


def test_random_numbers_at_the_ends(ctx):
    l = normal(6, 777, "f32", 4)
    token, _ = check(ctx, l, u=[0.0, 1 - 2.0 ** -24, 1.0, -0.5, 2.0, 1e-12])
    assert token[0] == 0 and token[3] == 0
    a = check(ctx, l[:1], u=[0.0])[0]
    b = torch.empty_like(a)
    aqmi.sample(ctx, l[:1], torch.full((1,), float("nan"), device="cuda"), b)
    assert torch.equal(a, b)


def test_greedy_takes_the_first_of_equals(ctx):
    l = normal(4, 5000, "bf16", 5)
    top = l.float().amax(1)
    for r in range(4):
        l[r, 4321] = l[r, 17 + r] = top[r].to(torch.bfloat16)
    token, logp = check(ctx, l, 0.0)
    first = [int((l[r].float() == top[r]).nonzero()[0]) for r in range(4)]
    assert token.tolist() == first and not logp.any()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V,ld", [(1000, 1003), (5001, 5003), (40001, 40003)])
def test_strided_rows(ctx, t, V, ld):
    full = normal(5, ld, t, V)
    full[:, V:] = 100.0   # not the row's
    check(ctx, full[:, :V], 0.8, 60, 0.9)
    check(ctx, full[:, :V], 1.0)


@pytest.mark.parametrize("V", [1, 64, 999, 5000])
def test_against_64_bits(ctx, V):
    l = normal(64, V, "f32", V, 2.0)
    t, k = 0.8, 20
    u = torch.rand(64, generator=torch.Generator().manual_seed(1)).cuda()
    for top_k in (None, torch.full((64,), k, dtype=torch.int32, device="cuda")):
        token, logp = torch.empty(64, dtype=torch.int32, device="cuda"), torch.empty(64, device="cuda")
        aqmi.sample(ctx, l, u, token, torch.full((64,), t, device="cuda"), top_k, logp=logp)
        e = (l.double() - l.double().amax(1, keepdim=True)).div(float(np.float32(t))).exp()
        if top_k is not None and k < V:
            e = torch.where(l >= l.topk(k, 1).values[:, -1:], e, 0)
        q = e / e.sum(1, keepdim=True)
        at = token.long()[:, None]
        hi = q.cumsum(1).gather(1, at).squeeze(1)
        lo = hi - q.gather(1, at).squeeze(1)
        assert bool(((lo - 2e-5 <= u) & (u <= hi + 2e-5)).all())
        ref = q.gather(1, at).squeeze(1).log()
        assert bool(((logp - ref).abs() <= 1.5e-5 + 2.0 ** -22 * ref.abs()).all())


def test_codes_of_a_frame_and_another_stream(ctx):
    """[B, Q] codes from [B, Q, N] logits, on a stream of its own."""
    l = normal(24, 512, "f32", 8)
    u = torch.rand(24, device="cuda")
    want = torch.empty(24, dtype=torch.int32, device="cuda")
    aqmi.sample(ctx, l, u, want)
    codes = torch.empty((3, 8), dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        aqmi.sample(ctx, l, u, codes)
    torch.cuda.synchronize()
    assert torch.equal(codes.flatten(), want)


def test_refusals(ctx):
    l, u = normal(4, 64, "f32", 1), torch.zeros(4, device="cuda")
    token = torch.empty(4, dtype=torch.int32, device="cuda")

    def call(t=0, l=l.data_ptr(), ld=64, rows=4, V=64, u=u.data_ptr(), token=token.data_ptr()):
        return ctx.lib.aq_sample(ctx.h, t, l, ld, rows, V, u, None, None, None, None, token, None)

    assert call() == 0 and call(rows=0, l=None, u=None, token=None) == 0
    for bad, status in [(dict(t=3), 1), (dict(t=-1), 1), (dict(l=None), 1), (dict(u=None), 1), (dict(token=None), 1),
                        (dict(ld=63), 2), (dict(rows=-1), 2), (dict(rows=(1 << 21) + 1), 2), (dict(V=0, ld=0), 2),
                        (dict(V=(1 << 20) + 1, ld=1 << 21), 2)]:
        assert call(**bad) == status, bad
        assert "aq_sample" in ctx.lib.aq_last_error(ctx.h).decode()
    with pytest.raises(ValueError):
        aqmi.sample(ctx, l, u[:3], token)
    with pytest.raises(ValueError):
        aqmi.sample(ctx, l, u, token, top_k=u)
    with pytest.raises(TypeError):
        aqmi.sample(ctx, l.double(), u, token)
