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
