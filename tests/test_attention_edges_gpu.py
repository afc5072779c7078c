"""aq_cross_attention and aq_prefix_attention where sizes, values and layouts meet a border."""

import pytest
import torch

import aqmi

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ctx():
    return aqmi.Context(0)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [1, 3, 33, 35, 64, 129, 250])
@pytest.mark.parametrize("T", [1, 40, 150])
def test_no_key_at_all(ctx, t, D, T):
    """Rows of zeros, and nothing beside them: not the columns behind a row, nor rows from q_len on."""
    B, H = 3, 2
    q = torch.ones((B, T, H, D), dtype=TYPES[t], device="cuda")
    none, no_prefix = q[:, :0, :1], q[0, :0, :1]
    rows = [T, 0, T // 2]
    q_len = torch.tensor(rows, dtype=torch.int32, device="cuda")
    for call in (lambda out: aqmi.prefix_attention(ctx, q, no_prefix, no_prefix, none, none, out, q_len=q_len),
                 lambda out: aqmi.cross_attention(ctx, q, none, none, out, q_len=q_len)):
        around = torch.full((B, T + 1, H, D + 9), 7.0, dtype=TYPES[t], device="cuda")
        call(around[:, :T, :, :D])
        want = torch.full_like(around, 7.0)
        for b in range(B):
            want[b, :rows[b], :, :D] = 0
        assert torch.equal(around, want)


FAR = {"f16": (4096.0, 2.0 ** 6), "bf16": (2.0 ** 24, 2.0 ** 18), "f32": (2.0 ** 24, 2.0 ** 8)}


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("scale", [2.0 ** -8, 1.0, 5.0, 1e37])
@pytest.mark.parametrize("B,T,P,S,D", [(1, 1, 0, 300, 64), (3, 5, 300, 40, 64), (2, 70, 90, 130, 128), (1, 1, 3000, 20, 128),
                                       (2, 140, 0, 300, 256)])
def test_scores_far_from_zero(ctx, t, sign, scale, B, T, P, S, D):
    """Scores of 2^30 (f16) and 2^54, exact in fp32, whose own rounding is far above what a weight may be off by: keys
    that are alike share the weight, and one that stands out takes all of it; at a scale of 1e37 the scores' products
    with it are beyond fp32."""
    size, step = FAR[t]
    H, Hkv, far = 4, 2, -1 if sign < 0 else 1
    kw = dict(dtype=TYPES[t], device="cuda")
    q = torch.full((B, T, H, D), size, **kw)
    k, pk = torch.full((B, S, Hkv, D), sign * size, **kw), torch.full((P, Hkv, D), sign * size, **kw)
    v, pv = torch.zeros((B, S, Hkv, D), **kw), torch.zeros((P, Hkv, D), **kw)
    v[:], pv[:] = torch.arange(S, device="cuda").remainder(8)[:, None, None], torch.arange(P, device="cuda").remainder(8)[:, None, None]
    u = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[t]
    own = S - T   # keys that every row sees
    out = torch.empty_like(q)

    def check(alone):
        """What each row gets: the mean over the keys that it sees, or the value of the one that stands out."""
        aqmi.prefix_attention(ctx, q, pk, pv, k, v, out, scale=scale)
        for i in sorted({0, T // 2, T - 1}):
            seen = torch.cat((pv.double(), v[0, :own + i + 1].double()))[:, 0, 0]
            want = (seen.mean() if alone is None else torch.tensor(float(alone))).item()
            # each rounding of a weight and of the output, and S + P fp32 additions to either sum
            assert bool(((out[:, i].double() - want).abs() <= want * (2 * u + (S + P) * 2.0 ** -22) + 1e-6).all()), i
        if P == 0 and T == 1:   # the same keys without an order
            crossed = torch.empty_like(q)
            aqmi.cross_attention(ctx, q, k, v, crossed, scale=scale)
            assert torch.equal(crossed, out)

    check(None)
    at = own // 3
    k[:, at] = sign * size + step   # the largest of all scores, by 2^24 and more
    v[:, at] = 5
    check(5)
    k[:, at] = sign * size
    k[:, :own] = sign * size - step   # far below the others: rows that see those give these nothing
    pk[:] = sign * size - step
    v[:, own:] = 3
    check(3)


def test_two_contexts_at_once():
    """Calls of two contexts on two streams, side by side on the device, each with parts in its own scratch."""
    g = torch.Generator().manual_seed(9)
    made = lambda *s: torch.randn(s, generator=g).bfloat16().cuda()
    work, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for B, P, S in ((40, 3000, 300), (3, 9000, 500)):
        q, k, v, pk, pv = made(B, 1, 8, 128), made(B, S, 2, 128), made(B, S, 2, 128), made(P, 2, 128), made(P, 2, 128)
        alone = torch.empty_like(q)
        context = aqmi.Context(0)
        aqmi.prefix_attention(context, q, pk, pv, k, v, alone)
        work.append((context, (q, pk, pv, k, v), alone, [torch.empty_like(q) for _ in range(20)]))
    torch.cuda.synchronize()
    for i in range(20):
        for stream, (context, inputs, _, outs) in zip(streams, work):
            with torch.cuda.stream(stream):
                aqmi.prefix_attention(context, *inputs, outs[i])
    torch.cuda.synchronize()
    for _, _, alone, outs in work:
        assert all(torch.equal(out, alone) for out in outs)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T", [1, 40, 150])
def test_subnormal_values(ctx, t, T):
    """The mean of equal values is that value: the weights' rounding is less than half a step of a 16-bit type's subnormal
    values; in f32 each of 300 products with a weight rounds to a multiple of 2^-149."""
    g = torch.Generator().manual_seed(T)
    for value in {"f16": (2.0 ** -24, 2.0 ** -15), "bf16": (2.0 ** -133, 2.0 ** -127), "f32": (2.0 ** -130, 2.0 ** -127)}[t]:
        q, k = (torch.randn((2, n, 2, 64), generator=g).to(TYPES[t]).cuda() for n in (T, 300))
        v, out = torch.full_like(k, value), torch.empty_like(q)
        aqmi.cross_attention(ctx, q, k, v, out)
        allowed = 300 * 2.0 ** -149 if t == "f32" else 0.0
        assert bool(((out.double() - value).abs() <= allowed).all())
