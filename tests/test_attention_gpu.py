"""aq_cross_attention and aq_prefix_attention against their definition in 64 bits.

Tolerances, from the arithmetic, per value, with W = sum p |v| / sum p:
  fp32 steps   a score is off by at most D 2^-24 scale sum |q k| (its products
               and sums) and its exponent's argument, a, by 2 * 2^-24 |a|; both
               change the weight by that share, above and below the line: twice;
               2^x by 2^-23, and a sum over S keys by S 2^-24, twice each
  16-bit types p is rounded once, half a step of its type: u W; the output once
               more, u |out| (and half of the least f16 step, 2^-25)
The errors of many values have either sign, so all of them together are held to
less: 2e-6 of the norm for fp32, and 1.25 u for the 16-bit types (each of the two
roundings has at most u / sqrt(3) in the mean)."""

import pytest
import torch

import aqmi

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # half a step


@pytest.fixture(scope="module")
def ctx():
    return aqmi.Context(0)


def made(g, t, *shape, mean=0.0):
    return (torch.randn(shape, generator=g) + mean).to(TYPES[t]).cuda()


def expected(q, k, v, sees, scale):
    """(out, W, allowed share) in 64 bits: q [T, H, D], k, v [S, Hkv, D] and which keys each row sees [T, S]."""
    q, k, v = (x.double().cpu() for x in (q, k, v))
    (T, H, D), (S, Hkv) = q.shape, k.shape[:2]
    k, v = (x.repeat_interleave(H // Hkv, 1).permute(1, 0, 2) for x in (k, v))   # [H, S, D]
    seen = sees.cpu().any(0)
    k, v = (torch.where(seen[:, None], x, torch.zeros((), dtype=torch.float64)) for x in (k, v))
    q = q.permute(1, 0, 2)
    z = (q @ k.transpose(1, 2) * scale).masked_fill(~sees.cpu(), -torch.inf)
    top = z.amax(2, keepdim=True) if S else torch.zeros((H, T, 1), dtype=torch.float64)
    a = z - torch.where(top > -torch.inf, top, 0.0)
    p = torch.exp(a)
    total = p.sum(2, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    size = (q.abs() @ k.abs().transpose(1, 2) * scale).masked_fill(~sees.cpu(), 0.0)
    size = size.amax(2, keepdim=True) if S else top
    # exponents below -40 are of weights below 2^-57: they count for nothing
    reach = 40.0
    share = 2 * (D * 2.0 ** -24 * size + 2 * 2.0 ** -24 * reach + 2.0 ** -23 + S * 2.0 ** -24)
    return tuple(x.permute(1, 0, 2) for x in (p @ v, p @ v.abs(), share.expand(H, T, D)))


def compare(got, parts, t):
    """got and what expected() gave for each of its streams' rows."""
    ref, W, share = (torch.cat([p[i] for p in parts]) for i in range(3))
    got = torch.cat(got).double().cpu()
    u = HALF[t]
    assert got.isfinite().all()
    assert bool(((got - ref).abs() <= (share + u) * W + (u + 2.0 ** -23) * ref.abs() + (2.0 ** -25 if t == "f16" else 1e-37)).all())
    assert (got - ref).norm() <= (1.25 * u if u else 2e-6) * ref.norm() + 1e-30


def check_cross(ctx, t, B, T, S, H, Hkv, D, lens=False, masked=0.0, scale=None, layout=None, seed=0, junk=True):
    g = torch.Generator().manual_seed(seed + 1000 * T + S)
    q, k, v = made(g, t, B, T, H, D), made(g, t, B, S, Hkv, D), made(g, t, B, S, Hkv, D, mean=0.25)
    q_len = kv_len = mask = None
    rows, keys = [T] * B, [S] * B
    sees = torch.ones((B, S), dtype=torch.bool)
    if lens:
        rows = [T - (3 * b) % (T + 1) for b in range(B)]
        keys = [max(0, S - (S * (5 * b % 8)) // 7) for b in range(B)]   # the whole and nothing among them
        q_len, kv_len = (torch.tensor(x, dtype=torch.int32).cuda() for x in (rows, keys))
        sees = torch.arange(S) < torch.tensor(keys)[:, None]
    if masked:
        mask = torch.rand((B, S), generator=g) >= masked
        mask[B // 2] &= B == 1
        sees = sees & mask
        mask = mask.cuda()
    if junk:   # what is left out does not matter
        for x, value in ((k, float("nan")), (v, float("inf"))):
            x[~sees.cuda()] = value
    out = torch.full_like(q, 7.0)
    if layout:
        q, k, v, out = (layout(x) for x in (q, k, v, out))
    aqmi.cross_attention(ctx, q, k, v, out, kv_len=kv_len, q_len=q_len, mask=mask, scale=scale)
    torch.cuda.synchronize()
    parts = [expected(q[b, :rows[b]], k[b], v[b], sees[b].expand(rows[b], S), D ** -0.5 if scale is None else scale)
             for b in range(B)]
    compare([out[b, :rows[b]] for b in range(B)], parts, t)
    for b in range(B):
        assert bool((out[b, rows[b]:] == 7).all())


def check_prefix(ctx, t, B, T, P, S, H, Hkv, D, lens=False, layout=None, seed=0):
    g = torch.Generator().manual_seed(seed + 1000 * T + S + P)
    q, k, v = made(g, t, B, T, H, D), made(g, t, B, S, Hkv, D), made(g, t, B, S, Hkv, D, mean=0.25)
    pk, pv = made(g, t, P, Hkv, D), made(g, t, P, Hkv, D, mean=0.25)
    q_len = kv_len = None
    rows, keys = [T] * B, [S] * B
    if lens:
        rows = [T - (3 * b) % (T + 1) for b in range(B)]
        keys = [max(0, S - (S * (5 * b % 8)) // 7) for b in range(B)]   # fewer keys than rows among them
        q_len, kv_len = (torch.tensor(x, dtype=torch.int32).cuda() for x in (rows, keys))
        for b in range(B):
            k[b, keys[b]:], v[b, keys[b]:] = float("nan"), float("nan")
    out = torch.full_like(q, 7.0)
    if layout:
        q, k, v, out = (layout(x) for x in (q, k, v, out))
    aqmi.prefix_attention(ctx, q, pk, pv, k, v, out, kv_len=kv_len, q_len=q_len)
    torch.cuda.synchronize()
    parts = []
    for b in range(B):
        own = torch.arange(S) <= keys[b] - rows[b] + torch.arange(rows[b])[:, None]
        sees = torch.cat((torch.ones((rows[b], P), dtype=torch.bool), own), 1)
        parts.append(expected(q[b, :rows[b]], torch.cat((pk, k[b])), torch.cat((pv, v[b])), sees, D ** -0.5))
    compare([out[b, :rows[b]] for b in range(B)], parts, t)
    for b in range(B):
        assert bool((out[b, rows[b]:] == 7).all())


def heads_first(x):
    return x.transpose(1, 2).contiguous().transpose(1, 2)


def off_by_one(x):
    """The same rows in memory that starts one element later, with odd strides."""
    B, n, H, D = x.shape
    wide = torch.zeros(B * (n + 1) * H * (D + 3) + 1, dtype=x.dtype, device=x.device)[1:].view(B, n + 1, H, D + 3)
    wide = wide[:, :n, :, :D]
    wide.copy_(x)
    return wide


CROSS = [(1, 1, 1, 1, 1, 1), (2, 1, 33, 4, 4, 64), (1, 3, 200, 6, 2, 80), (3, 37, 333, 6, 3, 100), (2, 130, 65, 2, 1, 128),
         (1, 40, 64, 8, 1, 33), (5, 2, 129, 4, 2, 256), (2, 70, 300, 3, 3, 200), (1, 1, 3000, 5, 1, 128), (4, 1, 1500, 8, 2, 64)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("B,T,S,H,Hkv,D", CROSS)
def test_cross(ctx, t, B, T, S, H, Hkv, D):
    check_cross(ctx, t, B, T, S, H, Hkv, D)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("masked", [0.0, 0.3])
@pytest.mark.parametrize("B,T,S,H,Hkv,D", CROSS[1:])
def test_cross_lengths_and_masks(ctx, t, masked, B, T, S, H, Hkv, D):
    """Streams without a key, rows that are left as they were, NaN and infinities in what is left out."""
    check_cross(ctx, t, B + 2, T, S, H, Hkv, D, lens=True, masked=masked)
    check_cross(ctx, t, B, T, S, H, Hkv, D, masked=0.5, scale=0.3)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layout", [heads_first, off_by_one])
@pytest.mark.parametrize("B,T,S,H,Hkv,D", [(2, 3, 70, 4, 2, 64), (2, 50, 130, 4, 2, 128), (3, 1, 600, 2, 2, 80), (1, 5, 90, 2, 1, 256)])
def test_cross_strides(ctx, t, layout, B, T, S, H, Hkv, D):
    check_cross(ctx, t, B, T, S, H, Hkv, D, lens=True, layout=layout)


PREFIX = [(1, 1, 1, 1, 1, 1, 1), (4, 1, 100, 33, 8, 2, 64), (3, 5, 77, 40, 6, 3, 100), (2, 150, 300, 200, 4, 2, 128),
          (40, 1, 700, 90, 4, 4, 128), (3, 20, 0, 300, 2, 1, 80), (2, 90, 0, 90, 2, 2, 64), (5, 3, 130, 70, 4, 1, 256),
          (1, 1, 5000, 1000, 4, 1, 128), (2, 40, 64, 40, 8, 1, 200), (3, 1, 40, 0, 2, 2, 64), (20, 2, 2500, 2, 2, 1, 33)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lens", [False, True])
@pytest.mark.parametrize("B,T,P,S,H,Hkv,D", PREFIX)
def test_prefix(ctx, t, lens, B, T, P, S, H, Hkv, D):
    check_prefix(ctx, t, B, T, P, S, H, Hkv, D, lens)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layout", [heads_first, off_by_one])
@pytest.mark.parametrize("B,T,P,S,H,Hkv,D", [(3, 4, 70, 40, 4, 2, 64), (2, 70, 130, 90, 4, 2, 128), (2, 3, 60, 50, 2, 1, 256)])
def test_prefix_strides(ctx, t, layout, B, T, P, S, H, Hkv, D):
    check_prefix(ctx, t, B, T, P, S, H, Hkv, D, True, layout)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("T", [9, 100])
def test_values_that_only_later_rows_see(ctx, t, D, value, T):
    """A value that is not finite in a causal key changes the rows that see it, and no row before."""
    g = torch.Generator().manual_seed(T)
    B, P, S, H = 2, 40, T + 13, 2
    q, k, v = made(g, t, B, T, H, D), made(g, t, B, S, H, D), made(g, t, B, S, H, D)
    pk, pv = made(g, t, P, H, D), made(g, t, P, H, D)
    at = 13 + T // 2   # the key of row T // 2
    for where in (k, v):
        clean, got = torch.empty_like(q), torch.empty_like(q)
        aqmi.prefix_attention(ctx, q, pk, pv, k, v, clean)
        kept = where[0, at, 1, 3].clone()
        where[0, at, 1, 3] = value
        aqmi.prefix_attention(ctx, q, pk, pv, k, v, got)
        where[0, at, 1, 3] = kept
        same = torch.ones((B, T, H, D), dtype=torch.bool)
        same[0, T // 2:, 1, :] = False
        assert torch.equal(got[same.cuda()], clean[same.cuda()])
        later = got[0, T // 2:, 1]
        if where is v:
            # only its column, and there the value itself where each weight is above 0
            assert torch.equal(later[:, [0, 1, 2, 4]].isfinite(), torch.ones_like(later[:, :4], dtype=torch.bool))
            want = torch.full_like(later[:, 3], value)
            assert bool(((later[:, 3] == want) | (later[:, 3].isnan() & (want.isnan() | (want == want)))).all())
            assert not later[:, 3].isfinite().any()
        elif value != value:
            assert later.isnan().all()


@pytest.mark.parametrize("t", TYPES)
def test_equal_scores_and_far_ones(ctx, t):
    """All keys alike: the mean of v.  One key far above the rest: its v, whatever the others."""
    q, k = torch.zeros((1, 3, 2, 64), dtype=TYPES[t], device="cuda"), torch.ones((1, 700, 2, 64), dtype=TYPES[t], device="cuda")
    v = torch.arange(700, device="cuda").view(1, 700, 1, 1).expand(1, 700, 2, 64).remainder(8).to(TYPES[t]).contiguous()
    out = torch.empty_like(q)
    aqmi.cross_attention(ctx, q, k, v, out)
    want = v.double().mean(1)[0, 0, 0].item()
    assert bool(((out.double() - want).abs() <= want * (HALF[t] * 2 + 1e-6)).all())
    q[:] = 60
    k[0, 411] = 60
    aqmi.cross_attention(ctx, q, k, v, out)
    assert bool((out == v[0, 411, 0, 0]).all())
    k.neg_()   # 699 keys alike, and one far below
    aqmi.cross_attention(ctx, q, k, v, out)
    want = (v.double().sum(1)[0, 0, 0] - v[0, 411, 0, 0].double()).item() / 699
    assert bool(((out.double() - want).abs() <= want * (HALF[t] * 2 + 1e-6)).all())


@pytest.mark.parametrize("t", TYPES)
def test_one_encoder_for_all_streams(ctx, t):
    g = torch.Generator().manual_seed(3)
    q, k, v = made(g, t, 6, 2, 4, 64), made(g, t, 1, 150, 2, 64), made(g, t, 1, 150, 2, 64)
    mask = torch.rand((1, 150), generator=g).cuda() < 0.5
    out, one = torch.empty_like(q), torch.empty_like(q)
    aqmi.cross_attention(ctx, q, k.expand(6, -1, -1, -1), v.expand(6, -1, -1, -1), out, mask=mask.expand(6, -1))
    aqmi.cross_attention(ctx, q, k.repeat(6, 1, 1, 1), v.repeat(6, 1, 1, 1), one, mask=mask.repeat(6, 1))
    assert torch.equal(out, one)


@pytest.mark.parametrize("T", [1, 60])
def test_out_may_be_q(ctx, T):
    g = torch.Generator().manual_seed(4)
    q, k, v = made(g, "bf16", 3, T, 4, 64), made(g, "bf16", 3, 900, 2, 64), made(g, "bf16", 3, 900, 2, 64)
    out = torch.empty_like(q)
    aqmi.cross_attention(ctx, q, k, v, out)
    aqmi.cross_attention(ctx, q, k, v, q)
    assert torch.equal(q, out)


@pytest.mark.parametrize("T", [1, 40])
def test_offsets_past_32_bits(ctx, T):
    """Keys 2^23 elements apart: the last of 600 starts past 2^32, and past 2^33 bytes."""
    g = torch.Generator().manual_seed(5)
    step, S, D = 1 << 23, 600, 64
    far = torch.empty(S * step, dtype=torch.bfloat16, device="cuda").view(1, S, 2, step // 2)
    k, v, q = made(g, "bf16", 1, S, 1, D), made(g, "bf16", 1, S, 1, D), made(g, "bf16", 1, T, 2, D)
    fk, fv = far[:, :, :1, :D], far[:, :, 1:, :D]
    fk.copy_(k)
    fv.copy_(v)
    out, want = torch.empty_like(q), torch.empty_like(q)
    aqmi.cross_attention(ctx, q, k, v, want)
    aqmi.cross_attention(ctx, q, fk, fv, out)
    assert torch.equal(out, want)
    aqmi.prefix_attention(ctx, q, k[0], v[0], k, v, want)
    aqmi.prefix_attention(ctx, q, fk[0], fv[0], fk, fv, out)
    assert torch.equal(out, want)


def test_lengths_outside_their_range(ctx):
    g = torch.Generator().manual_seed(6)
    q, k, v = made(g, "bf16", 4, 3, 2, 64), made(g, "bf16", 4, 50, 2, 64), made(g, "bf16", 4, 50, 2, 64)
    out, want = torch.zeros_like(q), torch.zeros_like(q)
    i32 = dict(dtype=torch.int32, device="cuda")
    aqmi.cross_attention(ctx, q, k, v, out, kv_len=torch.tensor([-5, 51, 1 << 30, 20], **i32), q_len=torch.tensor([3, 9, -1, 2], **i32))
    aqmi.cross_attention(ctx, q, k, v, want, kv_len=torch.tensor([0, 50, 50, 20], **i32), q_len=torch.tensor([3, 3, 0, 2], **i32))
    assert torch.equal(out, want) and not out[0].any() and not out[2].any()


def test_empty_calls(ctx):
    z = lambda *s: torch.zeros(s, device="cuda")
    for B, T, S in ((0, 1, 5), (2, 0, 5)):
        aqmi.cross_attention(ctx, z(B, T, 2, 64), z(B, S, 2, 64), z(B, S, 2, 64), z(B, T, 2, 64))
        aqmi.prefix_attention(ctx, z(B, T, 2, 64), z(3, 2, 64), z(3, 2, 64), z(B, S, 2, 64), z(B, S, 2, 64), z(B, T, 2, 64))
    out = torch.full((2, 3, 2, 64), 7.0, device="cuda")
    aqmi.cross_attention(ctx, z(2, 3, 2, 64), z(2, 0, 2, 64), z(2, 0, 2, 64), out)
    assert not out.any()
    out.fill_(7)
    aqmi.prefix_attention(ctx, z(2, 3, 2, 64), z(0, 2, 64), z(0, 2, 64), z(2, 0, 2, 64), z(2, 0, 2, 64), out)
    assert not out.any()


def test_refusals(ctx):
    lib = ctx.lib
    x = torch.zeros((2, 8, 4, 64), device="cuda")
    ok = aqmi.Heads(x.data_ptr(), 2048, 256, 64)
    null, back = aqmi.Heads(None, 2048, 256, 64), aqmi.Heads(x.data_ptr(), 2048, -256, 64)
    shared, closer = aqmi.Heads(x.data_ptr(), 0, 256, 64), aqmi.Heads(x.data_ptr(), 2048, 256, 63)

    def cross(t=0, B=2, T=8, S=8, H=4, Hkv=4, D=64, q=ok, k=ok, v=ok, mask=None, mask_ld=8, scale=0.1, out=ok):
        return lib.aq_cross_attention(ctx.h, t, B, T, S, H, Hkv, D, q, k, v, None, None, mask, mask_ld, scale, out)

    def prefix(t=0, B=2, T=8, P=8, S=8, H=4, Hkv=4, D=64, q=ok, pk=ok, pv=ok, k=ok, v=ok, scale=0.1, out=ok):
        return lib.aq_prefix_attention(ctx.h, t, B, T, P, S, H, Hkv, D, q, pk, pv, k, v, None, None, scale, out)

    assert cross() == 0 and prefix() == 0
    assert cross(B=0, q=null, k=null, v=null, out=null) == 0 and prefix(T=0, q=null, out=null) == 0
    common = [(dict(t=3), 1), (dict(t=5), 1), (dict(scale=0.0), 1), (dict(scale=-1.0), 1), (dict(scale=float("nan")), 1),
              (dict(scale=float("inf")), 1), (dict(q=null), 1), (dict(k=null), 1), (dict(v=null), 1), (dict(out=null), 1),
              (dict(B=-1), 2), (dict(T=-1), 2), (dict(S=-1), 2), (dict(S=(1 << 30) + 1), 2), (dict(H=0), 2), (dict(Hkv=0), 2),
              (dict(H=6), 2), (dict(D=0), 2), (dict(D=257), 2), (dict(B=1 << 20, T=1 << 20), 2), (dict(q=back), 2),
              (dict(k=back), 2), (dict(v=back), 2), (dict(out=back), 2), (dict(out=shared), 2), (dict(out=closer), 2)]
    for call, name, more in ((cross, "aq_cross_attention", [(dict(mask=x.data_ptr(), mask_ld=7), 2), (dict(mask=x.data_ptr(), mask_ld=-1), 2)]),
                             (prefix, "aq_prefix_attention", [(dict(P=-1), 2), (dict(P=(1 << 30) + 1), 2), (dict(pk=null), 1),
                                                              (dict(pv=null), 1), (dict(pk=back), 2), (dict(pv=back), 2)])):
        for bad, status in common + more:
            assert call(**bad) == status, (name, bad)
            assert name in lib.aq_last_error(ctx.h).decode()
    q, i32 = x.bfloat16(), torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (lambda: aqmi.cross_attention(ctx, x, x[:, :, :, :32], x, x), lambda: aqmi.cross_attention(ctx, x, x, x[:1], x),
                lambda: aqmi.cross_attention(ctx, x, x, x, x, kv_len=i32[:1]), lambda: aqmi.cross_attention(ctx, x, x, x, x, q_len=i32.long()),
                lambda: aqmi.cross_attention(ctx, x, x, x, x, mask=x[:, :, 0, 0]), lambda: aqmi.cross_attention(ctx, x, x.cpu(), x, x),
                lambda: aqmi.prefix_attention(ctx, x, x[0], x[0, :4], x, x, x)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: aqmi.cross_attention(ctx, x, q, x, x), lambda: aqmi.prefix_attention(ctx, x, x[0], x[0], x, x, q)):
        with pytest.raises(TypeError):
            bad()


def test_other_streams_and_captured_graphs(ctx):
    """Calls whose parts are joined share the context's scratch: on other streams, in two graphs, and with larger
    eager calls between their replays each gives the eager result."""
    g = torch.Generator().manual_seed(8)
    sets = []
    for B, P, S in ((2, 900, 700), (9, 3000, 300)):
        s = dict(q=made(g, "bf16", B, 1, 8, 128), pk=made(g, "bf16", P, 2, 128), pv=made(g, "bf16", P, 2, 128),
                 k=made(g, "bf16", B, S, 2, 128), v=made(g, "bf16", B, S, 2, 128))
        s["out"], s["cross"] = torch.empty_like(s["q"]), torch.empty_like(s["q"])
        s["len"] = torch.full((B,), S, dtype=torch.int32, device="cuda")
        sets.append(s)

    def work(s):
        aqmi.prefix_attention(ctx, s["q"], s["pk"], s["pv"], s["k"], s["v"], s["out"], kv_len=s["len"])
        aqmi.cross_attention(ctx, s["q"], s["k"], s["v"], s["cross"], kv_len=s["len"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for s in sets:
            work(s)
    torch.cuda.synchronize()
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            work(s)
    big = [made(g, "f32", 3, 1, 32, 128), made(g, "f32", 3, 9000, 32, 128)]
    for turn in range(3):
        aqmi.cross_attention(ctx, big[0], big[1], big[1], torch.empty_like(big[0]))
        for s in sets:
            s["q"].copy_(torch.randn(s["q"].shape, generator=g))
            s["len"].copy_(torch.randint(0, s["k"].shape[1] + 1, s["len"].shape, generator=g))
            work(s)
        want = [(s["out"].clone(), s["cross"].clone()) for s in sets]
        torch.cuda.synchronize()
        for s in sets:
            s["out"].fill_(7)
            s["cross"].fill_(7)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for s, w in zip(sets, want):
            assert torch.equal(s["out"], w[0]) and torch.equal(s["cross"], w[1])
