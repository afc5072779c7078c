"""The operators of a layer that answers with codes, as cases to measure.

Between the rows that the norm writes and the head that the sampling reads, a
decoder over this library's codes spends its time in three calls, the kinds
here:

  i8      y = W x + bias in 8-bit whole numbers, a scale for each row of x and
          each row of W; x comes in 8 bits with its scales (as the norm writes
          it), or in a floating type and is brought to 8 bits within the call
  cross   attention of a stream's rows to the states of an encoder, which have
          a length (and a mask) of their own
  prefix  causal attention of streams that share a long prefix (a voice
          prompt) held once, and go on from it with keys of their own

prepare() makes the inputs of a seed on the GPU; run() computes the plain form
in elementary torch operations or, where `own` is true, makes the library's
calls; exact() restates each definition in 64 bits.
"""

import math
import pathlib
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # The joint query, key and value projection of a 1024-wide model with
        # shared heads, one token, from the norm's row: pure latency.
        dict(name="i8_token", kind="i8", M=1, K=1024, N=1536, x="i8", bias=False, out="bf16"),
        # An odd-sized layer after an activation, which leaves floating rows.
        dict(name="i8_ragged", kind="i8", M=37, K=1001, N=2051, x="f32", bias=True, out="f32"),
        # A wide layer for 64 concurrent streams: bound by the weights' way
        # from memory.
        dict(name="i8_streams", kind="i8", M=64, K=8192, N=16384, x="bf16", bias=False, out="bf16"),
        # A long prefill: bound by the matrix instructions.
        dict(name="i8_prefill", kind="i8", M=16384, K=8192, N=8192, x="i8", bias=True, out="bf16"),
        # One token against a sentence of text: pure latency.
        dict(name="cross_token", kind="cross", B=1, T=1, H=16, Hkv=16, D=64, S=203, type="bf16", ragged=False, masked=0.0),
        # Clips of different lengths with holes, fp32, one of them empty.
        dict(name="cross_ragged", kind="cross", B=3, T=37, H=6, Hkv=2, D=80, S=333, type="f32", ragged=True, masked=0.2),
        # One token each of 64 streams over 30 s clips: bound by the keys' and
        # values' way from memory.
        dict(name="cross_streams", kind="cross", B=64, T=1, H=32, Hkv=8, D=128, S=1500, type="bf16", ragged=True,
             masked=0.0),
        # Whole answers scored against 30 s clips: bound by arithmetic.
        dict(name="cross_clips", kind="cross", B=8, T=4096, H=16, Hkv=16, D=128, S=1500, type="f16", ragged=False,
             masked=0.0),
        # A few takes of one sentence with one voice, a token each.
        dict(name="prefix_token", kind="prefix", B=4, T=1, H=16, Hkv=4, D=64, P=1499, S=101, type="bf16", ragged=False),
        # A short step of several tokens (drafts to be checked) in fp32.
        dict(name="prefix_ragged", kind="prefix", B=5, T=23, H=6, Hkv=3, D=100, P=701, S=211, type="f32", ragged=True),
        # A server's batch on one long prompt, a token each.
        dict(name="prefix_streams", kind="prefix", B=128, T=1, H=32, Hkv=8, D=128, P=16384, S=1024, type="bf16",
             ragged=True),
        # The batch's own prompts behind the shared one: bound by arithmetic.
        dict(name="prefix_prompts", kind="prefix", B=16, T=512, H=16, Hkv=4, D=128, P=8192, S=512, type="f16",
             ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(("i8", "cross", "prefix"))
    if kind == "i8":
        K, N = _log(rng, 64, 8192), _log(rng, 64, 16384)
        M = _log(rng, 1, min(16384, 10 ** 8 // N, 16384 * 8192 * 8192 // (K * N)))
        return dict(kind=kind, M=M, K=K, N=N, x=rng.choice(("i8", "i8", "f32", "f16", "bf16")), bias=rng.random() < 0.5,
                    out=rng.choice(tuple(TYPES)))
    Hkv, G, D = rng.choice((1, 2, 4, 6, 8, 16)), rng.choice((1, 1, 2, 4, 5, 8)), rng.choice((32, 64, 64, 80, 100, 128, 128, 256))
    H, t = Hkv * G, rng.choice(tuple(TYPES))
    room = 2 ** 24 * 32 // 10 // H  # pairs of rows and keys, heads apart; fp32 below takes a share of them
    room = room // 8 if t == "f32" else room
    T = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
    if kind == "cross":
        S = _log(rng, 1, min(16384, room // T))
        B = _log(rng, 1, max(1, min(128, room // (T * S), 2 ** 26 // (S * Hkv * D), 2 ** 26 // (T * H * D))))
        return dict(kind=kind, B=B, T=T, H=H, Hkv=Hkv, D=D, S=S, type=t, ragged=rng.random() < 0.5,
                    masked=rng.choice((0.0, 0.0, 0.3)))
    P = _log(rng, 1, max(1, min(32768, room // T - T)))
    S = T + _log(rng, 1, max(1, min(4096, room // T - P)))
    B = _log(rng, 1, max(1, min(128, room // (T * (P + S)), 2 ** 26 // (S * Hkv * D), 2 ** 26 // (T * H * D))))
    return dict(kind=kind, B=B, T=T, H=H, Hkv=Hkv, D=D, P=P, S=S, type=t, ragged=rng.random() < 0.5)


def _ramp(n, most, ragged):
    """n lengths up to `most`, of many sizes if ragged."""
    return [most - most * (5 * i % 8) // 11 if ragged else most for i in range(n)]


def _lengths(c):
    """(rows of each stream, keys of each): the same for every seed, so that work() knows them."""
    rows = [max(1, n) for n in _ramp(c["B"], c["T"], c["ragged"])]
    if c["kind"] == "cross":
        keys = _ramp(c["B"], c["S"], c["ragged"])
        if c["ragged"] and c["B"] > 2:
            keys[1] = 0  # a stream without a clip
        return rows, keys
    past = _ramp(c["B"], c["S"] - c["T"], c["ragged"])
    return rows, [r + p for r, p in zip(rows, past)]


def _inputs(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device=DEV)

    def whole(*shape):
        return torch.round(torch.clamp(127 / 3.5 * normal(*shape), -127, 127)).to(torch.int8)

    if c["kind"] == "i8":
        M, K, N = c["M"], c["K"], c["N"]
        s = dict(w=whole(N, K), scale=(0.5 + uniform(N)) * 3.5 / 127 / math.sqrt(K), bias=0.1 * normal(N) if c["bias"] else None)
        if c["x"] == "i8":
            return dict(s, x=whole(M, K), x_scale=(0.5 + uniform(M)) * 3.5 / 127)
        x = normal(M, K)
        x *= 1 + 6 * (uniform(K) < 0.01)  # a few channels stand out
        return dict(s, x=x.to(TYPES[c["x"]]), x_scale=None)
    t, B, T, H, Hkv, D, S = TYPES[c["type"]], *(c[k] for k in ("B", "T", "H", "Hkv", "D", "S"))
    rows, keys = _lengths(c)
    s = dict(q=(1.5 * normal(B, T, H, D)).to(t), k=normal(B, S, Hkv, D).to(t), v=(normal(B, S, Hkv, D) + 0.25).to(t),
             out=torch.zeros((B, T, H, D), dtype=t, device=DEV), q_len=None, kv_len=None, mask=None)
    if c["ragged"]:
        s.update(q_len=torch.tensor(rows, dtype=torch.int32, device=DEV), kv_len=torch.tensor(keys, dtype=torch.int32, device=DEV))
    if c["kind"] == "prefix":
        return dict(s, prefix_k=normal(c["P"], Hkv, D).to(t), prefix_v=(normal(c["P"], Hkv, D) + 0.25).to(t))
    if c["masked"]:
        s["mask"] = uniform(B, S) >= c["masked"]
        s["mask"][B // 2] &= B == 1  # of several streams one keeps nothing
    return s


_kept = {}


def _library():
    """The binding and a context, as a program holds them for its lifetime."""
    if not _kept:
        sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent / "audio.cpp_amd"))
        import aqmi

        _kept.update(aqmi=aqmi, ctx=aqmi.Context(0))
    return _kept["aqmi"], _kept["ctx"]


def prepare(case, seed):
    c = dict(case)
    s = dict(_inputs(c, seed), case=c)
    if own and c["kind"] == "i8":
        aqmi, ctx = _library()
        bias = None if s["bias"] is None else s["bias"].cpu().numpy()
        s["linear"] = aqmi.I8Linear(ctx, s["w"].cpu().numpy(), s["scale"].cpu().numpy(), bias)
    return s


# ---- the library's calls ----------------------------------------------------


def _own_i8(s, c):
    out = torch.empty((c["M"], c["N"]), dtype=TYPES[c["out"]], device=DEV)
    s["linear"].forward(s["x"], out, s["x_scale"])
    return out


def _own_cross(s, c):
    aqmi, ctx = _library()
    aqmi.cross_attention(ctx, s["q"], s["k"], s["v"], s["out"], kv_len=s["kv_len"], q_len=s["q_len"], mask=s["mask"])
    return s["out"]


def _own_prefix(s, c):
    aqmi, ctx = _library()
    aqmi.prefix_attention(ctx, s["q"], s["prefix_k"], s["prefix_v"], s["k"], s["v"], s["out"], kv_len=s["kv_len"],
                          q_len=s["q_len"])
    return s["out"]


# ---- the plain forms --------------------------------------------------------


def _plain_i8(s, c):
    x, scale = s["x"].float(), s["x_scale"]
    if scale is None:
        # in 64 bits: a value next to the middle of two whole numbers goes to one of them
        most = x.abs().amax(1, keepdim=True).double()
        x = torch.round(torch.where(most > 0, x.double() * 127 / most, 0)).float()
        scale = (most / 127).float().squeeze(1)
    y = x @ s["w"].float().t() * (scale[:, None] * s["scale"])
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(TYPES[c["out"]])


def _by_head(t, Hkv):
    """[B, T, H, D] as [B, Hkv, rows, D] in fp32, the rows of a head's group together."""
    B, T, H, D = t.shape
    return t.float().reshape(B, T, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)


def _softmax(scores):
    """(weights, their sums); a row without a key has none of either."""
    top = scores.amax(3, keepdim=True)
    e = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    return e, e.sum(3, keepdim=True)


def _joined(o, total, s, c):
    """[B, Hkv, rows, D] sums over their weights, as the outputs; rows past a stream's last keep what `out` holds."""
    B, T, H, D = s["q"].shape
    o = torch.where(total > 0, o / total, 0.0)
    o = o.reshape(B, c["Hkv"], H // c["Hkv"], T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(s["q"].dtype)
    if s["q_len"] is None:
        return o
    used = torch.arange(T, device=DEV) < s["q_len"][:, None]
    return torch.where(used[:, :, None, None], o, s["out"])


def _keys(s, c):
    """Which keys [B, S] a stream has."""
    seen = torch.ones((c["B"], c["S"]), dtype=torch.bool, device=DEV)
    if s["kv_len"] is not None:
        seen = torch.arange(c["S"], device=DEV) < s["kv_len"][:, None]
    return seen if s["mask"] is None else seen & s["mask"]


def _plain_cross(s, c):
    seen = _keys(s, c)[:, None, None, :]
    k, v = _by_head(s["k"], c["Hkv"]), _by_head(s["v"], c["Hkv"])
    scores = _by_head(s["q"], c["Hkv"]) @ k.transpose(2, 3).contiguous() / math.sqrt(c["D"])
    e, total = _softmax(scores.masked_fill_(~seen, -math.inf))
    return _joined(e @ torch.where(seen.transpose(2, 3), v, 0.0), total, s, c)


def _plain_prefix(s, c):
    B, T, H, D = s["q"].shape
    q, G = _by_head(s["q"], c["Hkv"]), H // c["Hkv"]
    rows = torch.full((B,), T, device=DEV) if s["q_len"] is None else s["q_len"]
    keys = torch.full((B,), c["S"], device=DEV) if s["kv_len"] is None else s["kv_len"]
    # row t sees the keys up to its own, which is rows - t before the stream's end
    last = (keys - rows)[:, None] + torch.arange(T, device=DEV)
    last = torch.where(torch.arange(T, device=DEV) < rows[:, None], last, -1).repeat(1, G)[:, None, :, None]
    k, v = _by_head(s["k"], c["Hkv"]), _by_head(s["v"], c["Hkv"])
    scores = torch.empty((B, c["Hkv"], G * T, c["P"] + c["S"]), device=DEV)
    scores[..., :c["P"]] = (q.transpose(0, 1).reshape(c["Hkv"], -1, D) @ s["prefix_k"].float().permute(1, 2, 0).contiguous()
                            ).reshape(c["Hkv"], B, G * T, -1).transpose(0, 1)
    scores[..., c["P"]:] = torch.where(torch.arange(c["S"], device=DEV) <= last, q @ k.transpose(2, 3).contiguous(), -math.inf)
    e, total = _softmax(scores.mul_(1 / math.sqrt(D)))
    o = e[..., :c["P"]].transpose(0, 1).reshape(c["Hkv"], B * G * T, -1) @ s["prefix_v"].float().transpose(0, 1).contiguous()
    o = o.reshape(c["Hkv"], B, G * T, D).transpose(0, 1) + e[..., c["P"]:] @ v
    return _joined(o, total, s, c)


def run(state):
    c = state["case"]
    if c["kind"] == "i8":
        return {"y": (_own_i8 if own else _plain_i8)(state, c)}
    if c["kind"] == "cross":
        return {"out": (_own_cross if own else _plain_cross)(state, c)}
    return {"out": (_own_prefix if own else _plain_prefix)(state, c)}


def work(case):
    c = case
    if c["kind"] == "i8":
        M, K, N = c["M"], c["K"], c["N"]
        moved = N * K + 4 * N * (2 if c["bias"] else 1) + M * N * TYPES[c["out"]].itemsize
        moved += M * (K + 4) if c["x"] == "i8" else M * K * TYPES[c["x"]].itemsize
        return {"bytes": moved, "flops": 2 * M * K * N}
    rows, keys = _lengths(c)
    t = TYPES[c["type"]].itemsize
    moved = t * 2 * sum(rows) * c["H"] * c["D"]
    if c["kind"] == "cross":
        kept = 1 - c["masked"]
        moved += t * 2 * int(kept * sum(keys)) * c["Hkv"] * c["D"] + (sum(keys) if c["masked"] else 0)
        pairs = int(kept * sum(r * k for r, k in zip(rows, keys)))
    else:
        moved += t * 2 * (c["P"] + sum(keys)) * c["Hkv"] * c["D"]
        pairs = sum(r * c["P"] + r * (k - r) + r * (r + 1) // 2 for r, k in zip(rows, keys))
    return {"bytes": moved, "flops": 4 * pairs * c["H"] * c["D"]}


# ---- the definitions in 64 bits -----------------------------------------------


def _exact_i8(s, c):
    x = s["x"].double()
    if s["x_scale"] is None:
        most = x.abs().max(dim=1, keepdim=True).values
        x, per = torch.nan_to_num(torch.round(127 * x / most)), most[:, 0] / 127
    else:
        per = s["x_scale"].double()
    y = torch.mm(s["w"].double(), x.t().contiguous()).t()
    y = y * per[:, None] * s["scale"].double()[None, :]
    return {"y": y if s["bias"] is None else y + s["bias"].double()}


def _exact_attention(s, c):
    rows, keys = _lengths(c)
    out, G = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV), c["H"] // c["Hkv"]
    for b in range(c["B"]):
        n, m = rows[b], keys[b]
        sees = torch.ones((n, m), dtype=torch.bool, device=DEV)
        if c["kind"] == "prefix":
            sees = torch.tril(sees, diagonal=m - n)
        elif s["mask"] is not None:
            sees &= s["mask"][b, :m]
        for h in range(c["Hkv"]):
            k, v, see = s["k"][b, :m, h].double(), s["v"][b, :m, h].double(), sees
            if c["kind"] == "prefix":
                k, v = torch.cat((s["prefix_k"][:, h].double(), k)), torch.cat((s["prefix_v"][:, h].double(), v))
                see = torch.cat((torch.ones((n, c["P"]), dtype=torch.bool, device=DEV), see), 1)
            for j in range(h * G, h * G + G):
                z = torch.mm(s["q"][b, :n, j].double(), k.t().contiguous()) / math.sqrt(c["D"])
                z[~see] = -math.inf
                p = torch.softmax(z, 1) if m or c["kind"] == "prefix" else z
                out[b, :n, j] = torch.mm(torch.nan_to_num(p), v)
    return {"out": out}


def exact(case, seed):
    c = dict(case)
    s = _inputs(c, int(seed))
    return _exact_i8(s, c) if c["kind"] == "i8" else _exact_attention(s, c)
