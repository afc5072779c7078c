"""The operators of a layer that answers with codes, together: the example's
steps against each operator's definition in 64 bits on its own inputs, and
captured in a HIP graph with the step that draws the codes.

Tolerances: an 8-bit product is a few fp32 roundings and one of its bf16 output,
2^-8 of the value; an attention is that twice (of the weights, which average to
at most one of the values' mean magnitude, and of the output), with the fp32
steps far below."""

import sys

import pytest
import torch

from conftest import ROOT

sys.path.insert(0, str(ROOT / "examples"))

import aqmi  # noqa: E402

pytestmark = pytest.mark.gpu


def dense(linear_seed):
    """The layer's matrices as the values that they stand for, in the order in which it makes them."""
    import code_layer as c
    import numpy as np

    rng = np.random.default_rng(linear_seed)
    got = []
    for out, width in (((c.HEADS + 2 * c.KV_HEADS) * c.HEAD, c.WIDTH), (c.WIDTH, c.HEADS * c.HEAD), (c.HEADS * c.HEAD, c.WIDTH),
                       (c.WIDTH, c.HEADS * c.HEAD)):
        w = rng.standard_normal((out, width), dtype=np.float32) / np.float32(np.sqrt(width))
        codes, scale = aqmi.i8_quantize(w)
        got.append(torch.from_numpy(codes).double() * torch.from_numpy(scale).double()[:, None])
    return got


def eight(x):
    """Rows as their 8-bit values stand for."""
    x = x.double()
    most = x.abs().amax(1, keepdim=True)
    return torch.round(x * 127 / most) * most / 127


def attention(q, k, v):
    """[H, D] over [n, Hkv, D] in 64 bits, and the mean magnitude of the values."""
    g = q.shape[0] // k.shape[1]
    k, v = (t.double().repeat_interleave(g, 1).permute(1, 0, 2) for t in (k, v))
    p = torch.softmax((k @ q.double()[:, :, None])[:, :, 0] / q.shape[1] ** 0.5, 1)[:, None]
    return (p @ v)[:, 0], (p @ v.abs())[:, 0]


def near(got, ref, extra=0.0, steps=1):
    got = got.double().cpu()
    assert bool(((got - ref).abs() <= 1.001 * 2.0 ** -8 * (ref.abs() + (steps - 1) * extra) + 1e-5).all())


@pytest.mark.parametrize("streams", [1, 5, 40])
def test_steps_of_the_example(streams):
    import code_layer as c

    layer = c.CodeLayer(aqmi.Context(0), streams, seed=3)
    w = dense(3)
    g = torch.Generator(device="cuda").manual_seed(streams)
    stream = torch.randn((streams, c.WIDTH), generator=g, device="cuda").bfloat16()
    kept = []
    for step in range(3):
        block = torch.randn((streams, c.WIDTH), generator=g, device="cuda").bfloat16()
        # the calls one by one, as step() makes them, with what each had
        seen = {}
        forward, prefix, cross = aqmi.I8Linear.forward, aqmi.prefix_attention, aqmi.cross_attention

        def watched(self, x, out, scale=None):
            forward(self, x, out, scale)
            seen[self] = (x.clone(), None if scale is None else scale.clone(), out.clone())

        def watched_prefix(ctx, q, *args, **kw):
            prefix(ctx, q, *args, **kw)
            seen["prefix"] = (q.clone(), args[4].clone())

        def watched_cross(ctx, q, *args, **kw):
            cross(ctx, q, *args, **kw)
            seen["cross"] = (q.clone(), args[2].clone())

        aqmi.I8Linear.forward, aqmi.prefix_attention, aqmi.cross_attention = watched, watched_prefix, watched_cross
        try:
            layer.step(stream, block)
        finally:
            aqmi.I8Linear.forward, aqmi.prefix_attention, aqmi.cross_attention = forward, prefix, cross
        torch.cuda.synchronize()
        for linear, matrix in zip((layer.qkv, layer.out, layer.text_q, layer.text_out), w):
            x, scale, out = seen[linear]
            x = eight(x.cpu()) if scale is None else x.cpu().double() * scale.cpu().double()
            near(out, x @ matrix.T)
        kept.append(seen[layer.qkv][2].view(streams, -1, c.HEAD)[:, c.HEADS:].cpu())
        own = torch.stack(kept, 1)   # [streams, tokens, key and value heads, D]
        for b in range(streams):
            k = torch.cat((layer.prompt_k.cpu(), own[b, :, :c.KV_HEADS]))
            v = torch.cat((layer.prompt_v.cpu(), own[b, :, c.KV_HEADS:]))
            ref, size = attention(seen["prefix"][0][b, 0].cpu(), k, v)
            near(seen["prefix"][1][b, 0], ref, size, 2)
            n = int(layer.text_len[b])
            ref, size = attention(seen["cross"][0][b, 0].cpu(), layer.text_k[b, :n].cpu(), layer.text_v[b, :n].cpu())
            near(seen["cross"][1][b, 0], ref, size, 2)
    assert layer.len.tolist() == [3] * streams


def test_captured_in_a_graph():
    """A layer and the drawing of its codes in one graph: replays with other calls between them equal the eager steps."""
    import code_layer as c

    ctx = aqmi.Context(0)
    layer, head = c.CodeLayer(ctx, 20), c.CodeStep(ctx, 20)
    g = torch.Generator(device="cuda").manual_seed(1)
    stream, block = (torch.randn((20, c.WIDTH), generator=g, device="cuda").bfloat16() for _ in range(2))
    u = torch.rand(20 * c.STAGES, generator=g, device="cuda")

    def work():
        head.draw(stream, layer.step(stream, block), u)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()   # the context's scratch grows here
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        work()
    other = [torch.randn((3, 1, 32, 128), device="cuda"), torch.randn((3, 4000, 32, 128), device="cuda")]
    for turn in range(4):
        new = [torch.randn((20, c.WIDTH), generator=g, device="cuda").bfloat16() for _ in range(2)]
        at = layer.len.clone()
        got = []
        for replayed in (True, False):
            stream.copy_(new[0])
            block.copy_(new[1])
            layer.len.copy_(at)
            torch.cuda.synchronize()
            if replayed:
                graph.replay()
            else:
                work()
            torch.cuda.synchronize()
            got.append([t.clone() for t in (stream, head.codes, head.logp, layer.block, layer.k, layer.v, layer.len)])
            aqmi.cross_attention(ctx, other[0], other[1], other[1], torch.empty_like(other[0]))   # takes more scratch
        for a, b in zip(*got):
            assert torch.equal(a, b)
