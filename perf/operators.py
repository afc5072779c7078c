"""The operators that answer with codes, as cases to measure.

A language model over this library's codes ends every step the same way: the
residual stream is added and normalised (and held in 8 bits with scales), a
matrix with 4-bit weights maps the row to logits, and a code is drawn from
each row of logits.  The kinds here are those three calls:

  norm    h = x + residual, y = h / rms(h) * weight, y in 8 bits with scales
          (whole numbers "i8", or "e4m3" floats)
  q4      y = W x + bias, W in 4 bits with a scale (and zero) per group, x in
          a floating type or in 8 bits with scales
  sample  one index per row of logits under temperature, top-k, top-p and
          min-p from a given random number

prepare() makes the inputs of a seed on the GPU; run() computes the plain form
in elementary torch operations or, where `own` is true, makes the library's
calls; exact() restates each definition in 64 bits.
"""

import math
import pathlib
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
EIGHT = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}
MOST = {"i8": 127.0, "e4m3": 448.0}  # the largest value of each
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # One token of one stream through a 1024-wide model: pure latency.
        dict(name="norm_token", kind="norm", M=1, D=1024, type="bf16", group=32, residual=True, y=False, q="e4m3"),
        # The frames of a 30 s clip in fp32 rows, a width off every tile, the
        # last group short, the row normalised and quantised together.
        dict(name="norm_ragged", kind="norm", M=1499, D=1001, type="f32", group=64, residual=True, y=True, q="i8"),
        # One scale per row and no 16-bit copy, a batch of prompts.
        dict(name="norm_batch", kind="norm", M=6000, D=4096, type="f16", group=0, residual=True, y=False, q="e4m3"),
        # A long prefill of a wide model: bound by memory.
        dict(name="norm_prefill", kind="norm", M=16384, D=8192, type="bf16", group=128, residual=True, y=True, q="e4m3"),
        # The code heads of a twelve-codebook model, one token: 12 x 1024
        # rows of logits from a bf16 hidden state.
        dict(name="q4_heads", kind="q4", M=1, K=1024, N=12288, group=32, x="bf16", x_group=0, zeros=False, bias=False,
             out="f32"),
        # An odd-sized projection of a few streams in fp32 with zero points.
        dict(name="q4_ragged", kind="q4", M=5, K=1000, N=4099, group=64, x="f32", x_group=0, zeros=True, bias=True,
             out="f32"),
        # Eight 2048-code heads for 64 concurrent streams.
        dict(name="q4_streams", kind="q4", M=64, K=4096, N=16384, group=128, x="f16", x_group=0, zeros=True, bias=False,
             out="f16"),
        # A wide layer, one token, the row already in 8 bits: bound by the
        # weights' way from memory.
        dict(name="q4_wide", kind="q4", M=1, K=8192, N=28672, group=128, x="i8", x_group=128, zeros=False, bias=False,
             out="bf16"),
        # One frame of twelve codes with the usual filters: pure latency.
        dict(name="sample_frame", kind="sample", rows=12, V=1024, type="f32", top_k=50, top_p=0.9, min_p=0.0,
             masked=0.0),
        # 64 streams x 8 codebooks, a part of each row masked, one row empty.
        dict(name="sample_streams", kind="sample", rows=512, V=2048, type="bf16", top_k=0, top_p=0.95, min_p=0.05,
             masked=0.25),
        # One token from a joint vocabulary of text and codes.
        dict(name="sample_text", kind="sample", rows=1, V=131071, type="f32", top_k=100, top_p=0.95, min_p=0.0,
             masked=0.0),
        # A full batch over such a vocabulary, nucleus only.
        dict(name="sample_batch", kind="sample", rows=256, V=160000, type="bf16", top_k=0, top_p=0.9, min_p=0.0,
             masked=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "q4", "sample"))
    if kind == "norm":
        D = _log(rng, 64, 8192)
        M = _log(rng, 1, min(16384, 16384 * 8192 // D))
        y, q = rng.choice(((True, ""), (True, "i8"), (True, "e4m3"), (False, "i8"), (False, "e4m3")))
        return dict(kind=kind, M=M, D=D, type=rng.choice(tuple(TYPES)), group=rng.choice((0, 32, 64, 128)) if q else 0,
                    residual=rng.random() < 0.8, y=y, q=q)
    if kind == "q4":
        x = rng.choice(("f32", "f16", "bf16", "i8", "e4m3"))
        group = rng.choice((32, 64, 128))
        K = _log(rng, 256, 8192)
        return dict(kind=kind, M=_log(rng, 1, 64), K=K, N=_log(rng, 256, min(28672, 16384 * 4096 // K)), group=group, x=x,
                    x_group=rng.choice((0, 32, 64, 128)) if x in EIGHT else 0, zeros=rng.random() < 0.5,
                    bias=rng.random() < 0.5, out=rng.choice(tuple(TYPES)))
    V = _log(rng, 256, 160000)
    return dict(kind=kind, rows=_log(rng, 1, min(512, 256 * 160000 // V)), V=V, type=rng.choice(tuple(TYPES)),
                top_k=rng.choice((0, 1, 20, 50, 400)), top_p=rng.choice((1.0, 0.5, 0.9, 0.99)),
                min_p=rng.choice((0.0, 0.02, 0.1)), masked=rng.choice((0.0, 0.0, 0.5)))


def _inputs(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device=DEV)

    if c["kind"] == "norm":
        t = TYPES[c["type"]]
        # The stream grows with depth and a few channels stand out.
        x = normal(c["M"], c["D"])
        x *= 1 + 6 * (uniform(c["D"]) < 0.01)
        return dict(x=x.to(t), residual=(2 * normal(c["M"], c["D"])).to(t) if c["residual"] else None,
                    weight=(1 + 0.2 * normal(c["D"])).to(t))
    if c["kind"] == "q4":
        M, K, N, G = c["M"], c["K"], c["N"], c["group"]
        groups = -(-K // G)
        s = dict(codes=torch.randint(0, 256, (N, -(-K // 2)), generator=g, device=DEV, dtype=torch.uint8),
                 scale=((0.5 + uniform(N, groups)) * (0.22 / math.sqrt(K))).to(torch.float16),
                 zero=torch.randint(4, 12, (N, groups), generator=g, device=DEV, dtype=torch.uint8) if c["zeros"] else None,
                 bias=0.1 * normal(N) if c["bias"] else None)
        if c["x"] in EIGHT:
            most = MOST[c["x"]]
            x = torch.clamp(most / 3.5 * normal(M, K), -most, most)
            s["x"] = (torch.round(x) if c["x"] == "i8" else x).to(EIGHT[c["x"]])
            s["x_scale"] = (0.5 + uniform(M, -(-K // c["x_group"]) if c["x_group"] else 1)) * 3.5 / most
        else:
            s["x"] = normal(M, K).to(TYPES[c["x"]])
        return s
    rows, V = c["rows"], c["V"]
    logits = 3 * normal(rows, V)
    if c["masked"]:
        logits[uniform(rows, V) < c["masked"]] = -math.inf
        if rows >= 16:
            logits[rows // 2] = -math.inf  # a row that its mask leaves empty
    temperature = 0.6 + 0.6 * uniform(rows)
    if rows >= 8:
        temperature[3] = 0  # a stream that asked for the most likely code
    return dict(logits=logits.to(TYPES[c["type"]]), temperature=temperature, u=uniform(rows),
                top_k=torch.full((rows,), c["top_k"], dtype=torch.int32, device=DEV) if c["top_k"] else None,
                top_p=torch.full((rows,), c["top_p"], device=DEV) if c["top_p"] < 1 else None,
                min_p=torch.full((rows,), c["min_p"], device=DEV) if c["min_p"] else None)


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
    if own and c["kind"] == "q4":
        aqmi, ctx = _library()
        host = {k: None if s[k] is None else s[k].cpu().numpy() for k in ("codes", "scale", "zero", "bias")}
        s["linear"] = aqmi.Q4Linear(ctx, host["codes"], host["scale"], c["K"], c["group"], host["zero"], host["bias"])
    return s


# ---- the library's calls ----------------------------------------------------


def _own_norm(s, c):
    aqmi, ctx = _library()
    x = s["x"]
    M, D = x.shape
    h = torch.empty_like(x)
    y = torch.empty_like(x) if c["y"] else None
    q = torch.empty((M, D), dtype=EIGHT[c["q"]], device=DEV) if c["q"] else None
    groups = -(-D // c["group"]) if c["group"] else 1
    scale = torch.empty((M, groups), dtype=torch.float32, device=DEV) if c["q"] else None
    aqmi.add_rmsnorm(ctx, x, s["weight"], EPS, residual=s["residual"], sum=h, y=y, q=q, scale=scale, group=c["group"])
    return h, y, q, scale


def _own_q4(s, c):
    out = torch.empty((c["M"], c["N"]), dtype=TYPES[c["out"]], device=DEV)
    if c["x"] in EIGHT:
        s["linear"].forward(s["x"], out, scale=s["x_scale"], group=c["x_group"])
    else:
        s["linear"].forward(s["x"], out)
    return out


def _own_sample(s, c):
    aqmi, ctx = _library()
    token = torch.empty(c["rows"], dtype=torch.int32, device=DEV)
    logp = torch.empty(c["rows"], dtype=torch.float32, device=DEV)
    aqmi.sample(ctx, s["logits"], s["u"], token, temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                min_p=s["min_p"], logp=logp)
    return token, logp


# ---- the plain forms --------------------------------------------------------


def _grouped(v, group):
    """[M, D] as [M, groups, group], the last group filled up with zeros."""
    M, D = v.shape
    group = group or D
    return torch.nn.functional.pad(v, (0, -D % group)).reshape(M, -1, group)


def _plain_norm(s, c):
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    v = h.float()
    y = v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * s["weight"].float()
    q = scale = None
    if c["q"]:
        g, most = _grouped(y, c["group"]), MOST[c["q"]]
        amax = g.abs().amax(2, keepdim=True)
        scale = (amax / most).squeeze(2)
        g = g * torch.where(amax > 0, most / amax, 0)
        g = torch.round(g) if c["q"] == "i8" else g
        q = g.reshape(c["M"], -1)[:, :c["D"]].to(EIGHT[c["q"]])
    return h, y.to(h.dtype) if c["y"] else None, q, scale


def _unpacked(s, c):
    """The weights [N, K] in fp32."""
    codes = torch.stack((s["codes"] & 15, s["codes"] >> 4), 2).reshape(c["N"], -1)[:, :c["K"]]
    at = torch.arange(c["K"], device=DEV) // c["group"]
    zero = 8.0 if s["zero"] is None else s["zero"].float()[:, at]
    return (codes.float() - zero) * s["scale"].float()[:, at]


def _plain_q4(s, c):
    x = s["x"].float()
    if c["x"] in EIGHT:
        at = torch.arange(c["K"], device=DEV) // (c["x_group"] or c["K"])
        x = x * s["x_scale"][:, at]
    y = x @ _unpacked(s, c).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(TYPES[c["out"]])


def _share(part, total):
    """floor(part * total / 2^24) for 0 <= part < 2^24 and whole total < 2^52."""
    hi, lo = total >> 26, total & ((1 << 26) - 1)
    return part * hi * 4 + ((part * lo) >> 24)


def _plain_sample(s, c):
    l = s["logits"].float()
    l = torch.where(torch.isnan(l), -math.inf, l)
    rows, V = l.shape
    greedy = ~(s["temperature"] > 0)
    top = l.amax(1, keepdim=True)
    # Weights relative to the most likely token, as whole numbers of 2^-31:
    # their sums do not depend on an order.
    per = torch.full_like(top, 1.4426950408889634) / torch.where(greedy, 1.0, s["temperature"])[:, None]
    z = torch.where(l == top, 0.0, l - top) * per
    e = torch.where(l > -math.inf, torch.exp2(z), 0.0)
    w = (e * 2.0 ** 31).to(torch.int64)
    # Top-k, then top-p of what top-k leaves, in order of the logits (the
    # lower index first where they are equal); min-p against the largest.
    order = torch.sort(l, dim=1, descending=True, stable=True).indices
    by = w.gather(1, order)
    rank = torch.arange(V, device=DEV)
    k = torch.full((rows, 1), V, device=DEV) if s["top_k"] is None else s["top_k"][:, None].long()
    k = torch.where(greedy[:, None], 1, torch.where(k <= 0, V, k))
    by = torch.where(rank < k, by, 0)
    if s["top_p"] is not None:
        p = (s["top_p"][:, None] * 2.0 ** 24).to(torch.int64)
        reach = by.cumsum(1)
        by = torch.where((reach - by < _share(p, reach[:, -1:])) | (rank == 0), by, 0)
    w = torch.zeros_like(w).scatter(1, order, by)
    if s["min_p"] is not None:
        w = torch.where(e >= s["min_p"][:, None], w, 0)
    reach = w.cumsum(1)
    total = reach[:, -1:]
    t = _share((s["u"][:, None] * 2.0 ** 24).to(torch.int64), total)
    token = (reach <= t).sum(1, keepdim=True)
    drawn = total > 0
    at = torch.where(drawn, token, 0)
    logp = z.gather(1, at) * 0.6931471805599453 - torch.log(total.float() * 2.0 ** -31)
    return (torch.where(drawn, token, -1).squeeze(1).to(torch.int32),
            torch.where(drawn, logp, -math.inf).squeeze(1))


def _stands(q, scale, c):
    """8 bits as the values they stand for: e4m3 is a floating type; the whole
    numbers are multiplied by their scales.  They have 7 bits and a sign, so
    bf16 holds them to half their own step."""
    if c["q"] == "e4m3":
        return q
    G = c["group"] or c["D"]
    out = torch.empty((c["M"], c["D"]), dtype=torch.bfloat16, device=DEV)
    if c["D"] % G:
        return torch.mul(q, scale[:, torch.arange(c["D"], device=DEV) // G], out=out)
    torch.mul(q.view(c["M"], -1, G), scale[:, :, None], out=out.view(c["M"], -1, G))
    return out


def run(state):
    c = state["case"]
    if c["kind"] == "norm":
        h, y, q, scale = (_own_norm if own else _plain_norm)(state, c)
        out = {"sum": h}
        if c["y"]:
            out["y"] = y
        if c["q"]:
            out["q"], out["scale"] = _stands(q, scale, c), scale
        return out
    if c["kind"] == "q4":
        return {"y": (_own_q4 if own else _plain_q4)(state, c)}
    token, logp = (_own_sample if own else _plain_sample)(state, c)
    return {"token": token, "logp": logp}


def work(case):
    c = case
    if c["kind"] == "norm":
        n, t = c["M"] * c["D"], TYPES[c["type"]].itemsize
        moved = n * t * (2 + c["residual"] + c["y"]) + c["D"] * t
        if c["q"]:
            moved += n + 4 * c["M"] * (-(-c["D"] // c["group"]) if c["group"] else 1)
        return {"bytes": moved, "flops": n * 6}
    if c["kind"] == "q4":
        M, K, N = c["M"], c["K"], c["N"]
        groups = -(-K // c["group"])
        moved = N * -(-K // 2) + N * groups * (3 if c["zeros"] else 2) + (4 * N if c["bias"] else 0)
        moved += M * N * TYPES[c["out"]].itemsize
        if c["x"] in EIGHT:
            moved += M * K + 4 * M * (-(-K // c["x_group"]) if c["x_group"] else 1)
        else:
            moved += M * K * TYPES[c["x"]].itemsize
        return {"bytes": moved, "flops": 2 * M * K * N}
    n = c["rows"] * c["V"]
    per_row = 4 * (4 + (c["top_k"] > 0) + (c["top_p"] < 1) + (c["min_p"] > 0))
    return {"bytes": n * TYPES[c["type"]].itemsize + c["rows"] * per_row, "flops": n * 5}


# ---- the definitions in 64 bits -----------------------------------------------


def _e4m3(v):
    """v rounded to the nearest e4m3 value, ties to the even one."""
    exponent = np.maximum(np.frexp(v)[1] - 1, -6)
    step = np.exp2(exponent - 3.0)
    return np.rint(v / step) * step


def _exact_norm(s, c):
    h = s["x"].double()
    if c["residual"]:
        h = (h + s["residual"].double()).to(s["x"].dtype).double()
    v, w = h.cpu().numpy(), s["weight"].double().cpu().numpy()
    root = np.sqrt(np.mean(np.square(v), axis=1) + EPS)
    y = v / root[:, None] * w
    out = {"sum": torch.from_numpy(v)}
    if c["y"]:
        out["y"] = torch.from_numpy(y)
    if c["q"]:
        starts = np.arange(0, c["D"], c["group"] or c["D"])
        per = np.maximum.reduceat(np.abs(y), starts, axis=1) / MOST[c["q"]]
        wide = np.repeat(per, np.diff(np.append(starts, c["D"])), axis=1)
        t = np.divide(y, wide, out=np.zeros_like(y), where=wide > 0)
        out["q"] = torch.from_numpy(_e4m3(t) if c["q"] == "e4m3" else np.rint(t) * wide)
        out["scale"] = torch.from_numpy(per)
    return out


def _exact_q4(s, c):
    def spread(v, group):  # one value per group, as one per column
        return v.double().repeat_interleave(group, 1)[:, :c["K"]]

    codes = torch.empty((c["N"], 2 * s["codes"].shape[1]), dtype=torch.float64, device=DEV)
    codes[:, 0::2] = (s["codes"] % 16).double()
    codes[:, 1::2] = torch.div(s["codes"], 16, rounding_mode="floor").double()
    w = codes[:, :c["K"]]
    w -= 8 if s["zero"] is None else spread(s["zero"], c["group"])
    w *= spread(s["scale"], c["group"])
    x = s["x"].double()
    if c["x"] in EIGHT:
        x = x * spread(s["x_scale"], c["x_group"] or c["K"])
    y = torch.mm(w, x.t().contiguous()).t()
    return {"y": y if s["bias"] is None else y + s["bias"].double()}


def _exact_sample(s, c):
    host = {k: None if s[k] is None else s[k].double().cpu().numpy()
            for k in ("logits", "temperature", "u", "top_k", "top_p", "min_p")}
    token, logp = np.full(c["rows"], -1, np.int32), np.full(c["rows"], -np.inf)
    for r, l in enumerate(host["logits"]):
        if not np.any(l > -np.inf):
            continue
        greedy = not host["temperature"][r] > 0
        z = (l - l.max()) / (math.log(2) * (1.0 if greedy else host["temperature"][r]))
        w = np.floor(np.exp2(z) * 2.0 ** 31)
        by = np.argsort(-l, kind="stable")
        count = 1 if greedy else c["V"] if host["top_k"] is None or host["top_k"][r] <= 0 else int(host["top_k"][r])
        by = by[:count]
        if host["top_p"] is not None and host["top_p"][r] < 1:
            before = np.cumsum(w[by]) - w[by]
            need = np.floor(np.floor(host["top_p"][r] * 2.0 ** 24) * (w[by].sum() / 2.0 ** 24))
            by = by[:max(1, np.searchsorted(before, need, side="left"))]
        kept = np.zeros_like(w)
        kept[by] = w[by]
        if host["min_p"] is not None:
            kept[np.exp2(z) < host["min_p"][r]] = 0
        reach = np.cumsum(kept)
        t = np.floor(np.floor(host["u"][r] * 2.0 ** 24) * (reach[-1] / 2.0 ** 24))
        token[r] = np.searchsorted(reach, t, side="right")
        logp[r] = z[token[r]] * math.log(2) - math.log(reach[-1] / 2.0 ** 31)
    return {"token": torch.from_numpy(token), "logp": torch.from_numpy(logp)}


def exact(case, seed):
    c = dict(case)
    s = _inputs(c, int(seed))
    return {"norm": _exact_norm, "q4": _exact_q4, "sample": _exact_sample}[c["kind"]](s, c)
