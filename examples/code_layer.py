"""A layer of a decoder over codes, for streams that speak different texts with
one voice, in front of the step that draws the codes (code_step.py).

  add_rmsnorm       the stream and the last block's output, normalised, in 8 bits
  I8Linear          query, key and value of the new token in one product
  prefix_attention  over the voice prompt, held once, and the stream's own tokens
  I8Linear          its output, brought to 8 bits row by row
  cross_attention   over the states of the stream's text
  CodeStep          heads, codes and latent

Random weights, so the sound is noise; the calls are the ones a server makes.
Run: python examples/code_layer.py [streams] [steps]
"""

from __future__ import annotations

import sys

import numpy as np
import torch

from code_step import STAGES, WIDTH, CodeStep, aqmi

HEADS, KV_HEADS, HEAD = 16, 4, 64
PROMPT, TEXT, TOKENS = 300, 80, 128   # keys of the voice prompt, of the longest text, and of a stream at most


class CodeLayer:
    """Weights, caches and buffers of `streams` streams; every call works in place."""

    def __init__(self, ctx: aqmi.Context, streams: int, seed: int = 0):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.ctx, self.streams = ctx, streams

        def linear(out, width):
            w = rng.standard_normal((out, width), dtype=np.float32) / np.float32(np.sqrt(width))
            return aqmi.I8Linear(ctx, *aqmi.i8_quantize(w))

        def half(*shape):
            return torch.randn(shape, generator=g, device="cuda").bfloat16()

        self.qkv = linear((HEADS + 2 * KV_HEADS) * HEAD, WIDTH)
        self.out = linear(WIDTH, HEADS * HEAD)
        self.text_q = linear(HEADS * HEAD, WIDTH)
        self.text_out = linear(WIDTH, HEADS * HEAD)
        self.norm = torch.ones(WIDTH, dtype=torch.bfloat16, device="cuda")
        # What a prompt pass has left: the voice's keys and values, and the texts'.
        self.prompt_k, self.prompt_v = half(PROMPT, KV_HEADS, HEAD), half(PROMPT, KV_HEADS, HEAD)
        self.text_k, self.text_v = half(streams, TEXT, HEADS, HEAD), half(streams, TEXT, HEADS, HEAD)
        self.text_len = torch.randint(1, TEXT + 1, (streams,), generator=g, device="cuda", dtype=torch.int32)
        self.k = torch.zeros((streams, TOKENS, KV_HEADS, HEAD), dtype=torch.bfloat16, device="cuda")
        self.v = torch.zeros_like(self.k)
        self.len = torch.zeros(streams, dtype=torch.int32, device="cuda")
        self.each = torch.arange(streams, device="cuda")
        self.q = torch.empty((streams, WIDTH), dtype=torch.int8, device="cuda")
        self.q_scale = torch.empty((streams, 1), device="cuda")
        self.heads = torch.empty((streams, 1, HEADS + 2 * KV_HEADS, HEAD), dtype=torch.bfloat16, device="cuda")
        self.text_heads = torch.empty((streams, 1, HEADS, HEAD), dtype=torch.bfloat16, device="cuda")
        self.seen = torch.empty_like(self.text_heads)
        self.block = torch.empty((streams, WIDTH), dtype=torch.bfloat16, device="cuda")

    def normalised(self, stream, block):
        """stream += block, and the row in 8 bits."""
        aqmi.add_rmsnorm(self.ctx, block, self.norm, 1e-6, residual=stream, sum=stream, q=self.q, scale=self.q_scale)

    def step(self, stream, block):
        """One token of each stream (of TOKENS at most: `len` is on the device and not looked at here); the block's
        output, not yet added to the stream."""
        self.normalised(stream, block)
        self.qkv.forward(self.q, self.heads.view(self.streams, -1), self.q_scale)
        at = self.len.long()
        self.k[self.each, at] = self.heads[:, 0, HEADS:HEADS + KV_HEADS]
        self.v[self.each, at] = self.heads[:, 0, HEADS + KV_HEADS:]
        self.len += 1
        aqmi.prefix_attention(self.ctx, self.heads[:, :, :HEADS], self.prompt_k, self.prompt_v, self.k, self.v, self.seen,
                              kv_len=self.len)
        self.out.forward(self.seen.view(self.streams, -1), self.block)
        self.normalised(stream, self.block)
        self.text_q.forward(self.q, self.text_heads.view(self.streams, -1), self.q_scale)
        aqmi.cross_attention(self.ctx, self.text_heads, self.text_k, self.text_v, self.seen, kv_len=self.text_len)
        self.text_out.forward(self.seen.view(self.streams, -1), self.block)
        return self.block


def main(streams: int = 4, steps: int = 8) -> None:
    if steps > TOKENS:
        raise ValueError(f"{steps} steps: a stream's caches hold {TOKENS} tokens")
    g = torch.Generator(device="cuda").manual_seed(0)
    ctx = aqmi.Context(0)
    layer, head = CodeLayer(ctx, streams), CodeStep(ctx, streams)
    stream = torch.randn((streams, WIDTH), generator=g, device="cuda").bfloat16()
    for i in range(steps):
        block = torch.randn((streams, WIDTH), generator=g, device="cuda").bfloat16()
        codes = head.draw(stream, layer.step(stream, block), torch.rand(streams * STAGES, generator=g, device="cuda"))
        latent = head.decode()
        print(f"step {i}: stream 0 codes {codes[0].tolist()}, |latent| {latent[0].norm().item():.2f}", flush=True)


if __name__ == "__main__":
    main(*map(int, sys.argv[1:3]))
