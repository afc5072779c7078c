"""The end of a step of a language model over codes: from the residual stream
to the next frame of codes, and from those to the latent that a decoder takes.

  add_rmsnorm   the stream and the last block's output, normalised, in 8 bits
  Q4Linear      one matrix with 4-bit weights for the heads of all codebooks
  sample        a code per codebook
  DacStages     the codes' latent (aq_dac_decode)

Random weights, so the sound is noise; the calls are the ones a server makes.
Run: python examples/code_step.py [streams] [steps]
"""

from __future__ import annotations

import pathlib
import sys

import numpy as np
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent / "audio.cpp_amd"))

import aqmi  # noqa: E402
from aqmi import synth  # noqa: E402

WIDTH, STAGES, CODES, LATENT = 1024, 12, 1024, 1024   # a 12-stage DAC under a 1024-wide model


class CodeStep:
    """Weights and buffers of `streams` streams; every call works in place."""

    def __init__(self, ctx: aqmi.Context, streams: int, seed: int = 0):
        rng = np.random.default_rng(seed)
        self.ctx, self.streams = ctx, streams
        heads = rng.standard_normal((STAGES * CODES, WIDTH), dtype=np.float32) * (3 / np.sqrt(WIDTH))
        codes, scale, zero = aqmi.q4_quantize(heads.astype(np.float32), 64, zeros=True)
        self.heads = aqmi.Q4Linear(ctx, codes, scale, WIDTH, 64, zero)
        w = synth.dac_weights(seed, STAGES, LATENT, CODES, bias=True)
        self.dac = aqmi.DacStages(ctx, w["w_in"], w["b_in"], w["codebook"], w["w_out"], w["b_out"])
        self.norm = torch.ones(WIDTH, dtype=torch.bfloat16, device="cuda")
        rows = streams * STAGES
        self.q = torch.empty((streams, WIDTH), dtype=torch.int8, device="cuda")
        self.q_scale = torch.empty((streams, WIDTH // 32), device="cuda")
        self.logits = torch.empty((streams, STAGES * CODES), device="cuda")
        self.codes = torch.empty((streams, STAGES), dtype=torch.int32, device="cuda")
        self.logp = torch.empty(rows, device="cuda")
        self.latent = torch.empty((streams, LATENT), device="cuda")
        self.temperature = torch.full((rows,), 0.9, device="cuda")
        self.top_k = torch.full((rows,), 50, dtype=torch.int32, device="cuda")
        self.top_p = torch.full((rows,), 0.95, device="cuda")

    def draw(self, stream, block, u):
        """stream += block; codes [streams, STAGES] drawn with u [streams * STAGES]."""
        aqmi.add_rmsnorm(self.ctx, block, self.norm, 1e-6, residual=stream, sum=stream, q=self.q, scale=self.q_scale,
                         group=32)
        self.heads.forward(self.q, self.logits, self.q_scale, 32)
        aqmi.sample(self.ctx, self.logits.view(-1, CODES), u, self.codes, self.temperature, self.top_k, self.top_p,
                    logp=self.logp)
        return self.codes

    def decode(self):
        """The latent of the frame drawn last."""
        self.dac.decode(self.codes, self.latent)
        return self.latent


def main(streams: int = 4, steps: int = 8) -> None:
    g = torch.Generator(device="cuda").manual_seed(0)
    step = CodeStep(aqmi.Context(0), streams)
    stream = torch.randn((streams, WIDTH), generator=g, device="cuda").bfloat16()
    for i in range(steps):
        block = torch.randn((streams, WIDTH), generator=g, device="cuda").bfloat16()
        codes = step.draw(stream, block, torch.rand(streams * STAGES, generator=g, device="cuda"))
        latent = step.decode()
        print(f"step {i}: stream 0 codes {codes[0].tolist()}, |latent| {latent[0].norm().item():.2f}", flush=True)


if __name__ == "__main__":
    main(*map(int, sys.argv[1:3]))
