"""Calls of one Context on several streams: the binding orders them, since
they share scratch.  The first tests run it over stand-ins for torch's
streams, without a GPU."""

import contextlib

import numpy as np
import pytest

import aqmi


class Stream:
    def __init__(self, cuda, raw):
        self.cuda, self.cuda_stream, self.capturing, self.gone = cuda, raw, False, False

    def wait_stream(self, other):
        if other.gone:
            raise RuntimeError("invalid resource handle")
        self.cuda.waits.append((self.cuda_stream, other.cuda_stream))


class Cuda:
    def __init__(self):
        self.waits, self.synchronized = [], 0
        self.now = self.default = Stream(self, 0)

    def current_stream(self, device):
        return self.now

    def is_current_stream_capturing(self):
        if self.now.gone:
            raise RuntimeError("invalid resource handle")
        return self.now.capturing

    def synchronize(self, device):
        self.synchronized += 1

    @contextlib.contextmanager
    def stream(self, s):
        before, self.now = self.now, s
        try:
            yield
        finally:
            self.now = before

    def is_available(self):
        return True


class Library:
    def __init__(self):
        self.streams = []

    def aq_ctx_create(self, device, stream, out):
        return 0

    def aq_ctx_set_stream(self, h, raw):
        self.streams.append(raw)
        return 0

    def aq_ctx_destroy(self, h):
        return 0


@pytest.fixture
def fake(monkeypatch):
    import sys
    import types

    torch = types.ModuleType("torch")
    torch.cuda, torch._C = Cuda(), types.SimpleNamespace()
    monkeypatch.setitem(sys.modules, "torch", torch)
    ctx = aqmi.Context(0, Library())
    return ctx, torch.cuda, lambda raw: Stream(torch.cuda, raw)


def test_a_change_of_stream_waits(fake):
    ctx, cuda, stream = fake
    a, b = stream(11), stream(22)
    ctx.use_current_stream()
    for s in (a, a, b):
        with cuda.stream(s):
            ctx.use_current_stream()
    ctx.use_current_stream()
    assert cuda.waits == [(11, 0), (22, 11), (0, 22)] and ctx.lib.streams == [0, 11, 11, 22, 0]


def test_captured_calls_neither_wait_nor_are_waited_for(fake):
    ctx, cuda, stream = fake
    a, g = stream(11), stream(33)
    with cuda.stream(a):
        ctx.use_current_stream()
    g.capturing = True
    with cuda.stream(g):
        ctx.use_current_stream()
        ctx.use_current_stream()
    assert cuda.waits == [(11, 0)] and ctx.lib.streams[-1] == 33
    ctx.use_current_stream()   # behind the last call that runs
    assert cuda.waits == [(11, 0), (0, 11)] and ctx.lib.streams[-1] == 0
    g.capturing = False
    with cuda.stream(g):       # its stream without the capture
        ctx.use_current_stream()
        g.capturing = True     # and a call elsewhere while it captures again
        ctx.use_current_stream()
        with cuda.stream(a):
            ctx.use_current_stream()
    assert cuda.waits == [(11, 0), (0, 11), (33, 0)] and ctx.lib.streams[-1] == 11


def test_a_stream_that_is_no_more(fake):
    ctx, cuda, stream = fake
    a = stream(11)
    with cuda.stream(a):
        ctx.use_current_stream()
    a.gone = True
    ctx.use_current_stream()
    assert cuda.synchronized == 1 and ctx.lib.streams[-1] == 0
    ctx.use_current_stream()
    assert cuda.synchronized == 1


@pytest.mark.gpu
def test_calls_on_two_streams():
    """Two products that share scratch, on streams with nothing between them
    but the context: the second one's end is behind the first one's, and both
    results are those of calls alone."""
    import torch

    ctx = aqmi.Context(0)
    r = np.random.default_rng(1)
    N, K, M = 512, 2048, 48
    lin = aqmi.Q4Linear(ctx, r.integers(0, 256, (N, K // 2), dtype=np.uint8),
                        r.uniform(0.01, 0.02, (N, K // 64)).astype(np.float16), K, 64)
    g = torch.Generator(device="cuda").manual_seed(1)
    xs = [torch.randn((M, K), generator=g, device="cuda").half() for _ in range(2)]
    want = [torch.empty((M, N), device="cuda") for _ in range(2)]
    for x, w in zip(xs, want):
        lin.forward(x, w)
    got = [torch.zeros((M, N), device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    ends = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    torch.cuda.synchronize()
    for rep in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                if i == 0:
                    torch.cuda._sleep(20_000_000)   # the first stream is busy meanwhile
                lin.forward(xs[i], got[i])
                ends[i].record()
        torch.cuda.synchronize()
        assert ends[0].elapsed_time(ends[1]) >= 0
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
