"""aq_i8_forward at sizes that the larger kinds of blocks take, with remainders on every side, and where the rows of x
are packed in several turns.  Tolerances as in test_i8_gpu.py; of the largest calls some rows are compared, those next
to a border among them."""

import numpy as np
import pytest
import torch

import aqmi
from test_i8_gpu import OUT, TYPES, matrix, reference, rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return aqmi.Context(0)


def check(ctx, N, K, M, t, out="f32", x_ld=None, y_ld=None, shift=0, some=None):
    """shift: x starts so many elements into its memory.  some: the rows to compare (None: all)."""
    w, scale, b = matrix(N, K, True, N + K)
    lin = aqmi.I8Linear(ctx, w, scale, b)
    x, s = rows(M, K, t, M, x_ld)
    if shift:
        moved = torch.zeros(x.numel() + shift, dtype=x.dtype, device="cuda")[shift:].view(M, K)
        moved.copy_(x)
        x = moved
    full = torch.full((M + 1, y_ld or N), 7.0, dtype=TYPES[out], device="cuda")
    lin.forward(x, full[:M, :N], s)
    torch.cuda.synchronize()
    at = torch.arange(M) if some is None else torch.tensor(sorted(set(some)))
    product, ref = reference(w, scale, b, x[at.cuda()], None if s is None else s[at.cuda()])
    got = full[at.cuda(), :N].double().cpu().numpy()
    allowed = 3e-7 * (np.abs(product) + np.abs(ref)) + OUT[out] * np.abs(ref) + (2.0 ** -25 if out == "f16" else 0)
    assert np.all(np.abs(got - ref) <= allowed)
    assert bool((full[:, N:] == 7).all()) and bool((full[M] == 7).all())
    return full[:M, :N]


@pytest.mark.parametrize("t,K,x_ld,shift", [("i8", 336, None, 0), ("i8", 336, 352, 0), ("i8", 336, None, 1), ("i8", 1001, 1003, 0),
                                            ("f32", 336, None, 0), ("f16", 1001, None, 3), ("bf16", 336, 340, 0)])
@pytest.mark.parametrize("out", OUT)
def test_blocks_of_256_by_256(ctx, t, K, x_ld, shift, out):
    """13 x 17 blocks, the last of 18 of 256 rows of W and of 4 of 256 rows of x."""
    check(ctx, 3090, K, 4100, t, out, x_ld, 3091 if out == "f32" else None, shift, [*range(0, 4100, 37), *range(4090, 4100)])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M", [33, 37, 64, 70])
def test_four_tiles_by_64_rows(ctx, t, M):
    """257 blocks of eight waves, and of four from 65 rows on; the last tile has 13 of 16 rows of W."""
    check(ctx, 16397, 1100, M, t, "f32" if M % 2 else "bf16", y_ld=16400)


@pytest.mark.parametrize("t", TYPES)
def test_rows_packed_in_turns(ctx, t):
    """64 MB are 8256 rows of 8100 columns: a second turn of nine rows goes to another kernel, with its own rows of x, of
    scales and of y; the same rows alone give the same bits."""
    N, K, M, turn = 300, 8100, 8265, 8256
    w, scale, b = matrix(N, K, True, N + K)
    y = check(ctx, N, K, M, t, some=[*range(0, M, 97), *range(turn - 5, M)])
    lin = aqmi.I8Linear(ctx, w, scale, b)
    x, s = rows(M, K, t, M)
    alone = torch.empty((M - turn, N), device="cuda")
    lin.forward(x[turn:], alone, None if s is None else s[turn:])
    assert torch.equal(alone, y[turn:])


def test_a_chunk_of_rows_does_not_see_another(ctx):
    """One row of values that are not finite is one row of NaN, wherever it lies among the turns."""
    N, K, M = 20, 8100, 8300
    w, scale, b = matrix(N, K, False, 1)
    lin = aqmi.I8Linear(ctx, w, scale, b)
    x, _ = rows(M, K, "bf16", 2)
    clean, got = (torch.empty((M, N), device="cuda") for _ in range(2))
    lin.forward(x, clean)
    for row in (0, 8255, 8256, 8299):
        kept = x[row, K - 1].clone()
        x[row, K - 1] = float("inf")
        lin.forward(x, got)
        x[row, K - 1] = kept
        assert got[row].isnan().all()
        got[row] = clean[row]
        assert torch.equal(got, clean)
