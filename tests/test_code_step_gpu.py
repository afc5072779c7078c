"""The operators that answer with codes, together: the example's step against
the same step in 64 bits from each operator's own inputs, and captured in a
HIP graph."""

import sys

import numpy as np
import pytest
import torch

from conftest import ROOT

sys.path.insert(0, str(ROOT / "examples"))

import aqmi  # noqa: E402

pytestmark = pytest.mark.gpu


def inputs(streams, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    import code_step

    return (torch.randn((streams, code_step.WIDTH), generator=g, device="cuda").bfloat16(),
            torch.randn((streams, code_step.WIDTH), generator=g, device="cuda").bfloat16(),
            torch.rand(streams * code_step.STAGES, generator=g, device="cuda"))


@pytest.mark.parametrize("streams", [1, 5, 40])
def test_step_of_the_example(streams):
    import code_step

    step = code_step.CodeStep(aqmi.Context(0), streams)
    stream, block, u = inputs(streams, streams)
    want = stream + block
    codes = step.draw(stream, block, u)
    latent = step.decode()
    torch.cuda.synchronize()
    assert torch.equal(stream, want)
    # The logits that the 8-bit row and the weights stand for.
    x = step.q.double() * step.q_scale.double().repeat_interleave(32, 1)
    y = want.double() / (want.double().square().mean(1, keepdim=True) + 1e-6).sqrt()
    # half a step of each group's scale, and what fp32 adds to it
    assert bool(((x - y).abs() <= 0.5001 * step.q_scale.double().repeat_interleave(32, 1)).all())
    # Each drawn code is one that the filters keep, and its latent the sum of its stages' tables.
    rows = step.logits.view(-1, code_step.CODES)
    kth = rows.topk(50, 1).values[:, -1:]
    assert bool((rows.gather(1, codes.view(-1, 1).long()) >= kth).all())
    again = torch.empty_like(latent)
    step.dac.decode(codes.clone(), again)
    assert torch.equal(latent, again) and bool(step.logp.isfinite().all())


def test_captured_in_a_graph():
    """Replays with other calls between them equal the eager step, each time."""
    import code_step

    step = code_step.CodeStep(aqmi.Context(0), 20)
    long_logits = torch.randn(6, 30000, device="cuda")
    long_u = torch.rand(6, device="cuda")
    top_p = torch.full((6,), 0.9, device="cuda")
    token = torch.empty(6, dtype=torch.int32, device="cuda")
    stream, block, u = inputs(20, 1)

    def work():
        step.draw(stream, block, u)
        aqmi.sample(step.ctx, long_logits, long_u, token, top_p=top_p)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()   # the context's scratch grows here
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        work()
    for seed in range(4):
        new_stream, new_block, new_u = inputs(20, 10 + seed)
        long_logits.normal_()
        stream.copy_(new_stream)
        block.copy_(new_block)
        u.copy_(new_u)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (stream, step.codes, step.logp, step.logits, token)]
        stream.copy_(new_stream)
        work()
        torch.cuda.synchronize()
        for a, b in zip(got, (stream, step.codes, step.logp, step.logits, token)):
            assert torch.equal(a, b)


def test_graph_keeps_its_scratch():
    """A later call that needs more scratch leaves a captured one what it uses."""
    ctx = aqmi.Context(0)
    g = torch.Generator(device="cuda").manual_seed(5)
    logits = 3 * torch.randn((3, 9000), generator=g, device="cuda")
    u, top_p = torch.rand(3, generator=g, device="cuda"), torch.full((3,), 0.95, device="cuda")
    token = torch.empty(3, dtype=torch.int32, device="cuda")
    r = np.random.default_rng(5)
    linears = [aqmi.Q4Linear(ctx, r.integers(0, 256, (n, k // 2), dtype=np.uint8),
                             r.uniform(0.01, 0.02, (n, k // 64)).astype(np.float16), k, 64) for n, k in ((96, 256), (64, 2048))]
    x, y = torch.randn((20, 256), generator=g, device="cuda").half(), torch.empty((20, 96), device="cuda")

    def work():
        linears[0].forward(x, y)
        aqmi.sample(ctx, logits, u, token, top_p=top_p)

    def larger():
        aqmi.sample(ctx, 3 * torch.randn((40, 50000), generator=g, device="cuda"), torch.rand(40, device="cuda"),
                    torch.empty(40, dtype=torch.int32, device="cuda"), top_p=torch.full((40,), 0.9, device="cuda"))
        linears[1].forward(torch.randn((200, 2048), generator=g, device="cuda").half(),
                           torch.empty((200, 64), device="cuda"))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    want = token.clone(), y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        work()
    for _ in range(3):
        larger()
        torch.cuda.synchronize()
        fill = [torch.full((1 << 20,), -1, dtype=torch.int32, device="cuda") for _ in range(8)]
        torch.cuda.synchronize()
        token.fill_(-7)
        y.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(token, want[0]) and torch.equal(y, want[1])
        assert all(bool((f == -1).all()) for f in fill)
