"""The scales of aq_add_rmsnorm where all but their own roundings are exact.

Half of a row's values are +-a and half +-b with (a^2 + b^2) / 2 = c^2 (all
whole, times a power of two), the row's length is a power of two and eps is 0:
the sum of squares, the mean and the root c are exact, and so is c * L (L = 127
or 448).  The scale of a group whose largest magnitude is b is then b / (c L)
rounded once, with no tolerance."""

import numpy as np
import pytest
import torch

import aqmi

pytestmark = pytest.mark.gpu

TRIPLES = [(1, 7, 5), (7, 17, 13), (7, 23, 17), (17, 31, 25), (1, 41, 29), (23, 47, 37)]


@pytest.fixture(scope="module")
def ctx():
    return aqmi.Context(0)


@pytest.mark.parametrize("t", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dt,most", [(torch.int8, 127), (torch.float8_e4m3fn, 448)])
@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("D", [128, 1024, 4096, 65536])
def test_rounded_once(ctx, t, dt, most, group, D):
    g = torch.Generator().manual_seed(D)
    rows, want = [], []
    for i, (a, b, c) in enumerate(TRIPLES):
        # b alone in the first half of the groups, a alone in the rest
        v = torch.cat((torch.full((D // 2,), float(b)), torch.full((D // 2,), float(a)))) * 2.0 ** (i - 3)
        rows.append(v * (2 * torch.randint(0, 2, (D,), generator=g) - 1))
        first = D // 2 // group if group else 1
        want.append([np.float32(b / (c * most))] * first + [np.float32(a / (c * most))] * (first if group else 0))
    x = torch.stack(rows).to(t).cuda()
    q = torch.empty(x.shape, dtype=dt, device="cuda")
    scale = torch.empty((len(TRIPLES), D // group if group else 1), device="cuda")
    aqmi.add_rmsnorm(ctx, x, None, 0.0, q=q, scale=scale, group=group)
    assert np.array_equal(scale.cpu().numpy(), np.array(want, np.float32))


@pytest.mark.parametrize("D", [64, 1024, 8192, 65536])
def test_root_within_half_a_unit(ctx, D):
    """Rows of one power of two: with an eps that is a multiple of 2^-10 the
    mean is exact, and y is 1 / root times that power.  The root's reciprocal
    is 2^-24 of itself off at most, and little more than half a unit means a
    hundredth beyond that."""
    h = torch.tensor([0.5, 1.0, 8.0], device="cuda")
    x = h[:, None].expand(3, D).contiguous()
    y = torch.empty_like(x)
    for k in range(1, 200):
        aqmi.add_rmsnorm(ctx, x, None, k * 2.0 ** -10, y=y)
        ref = h.double() / (h.double().square() + k * 2.0 ** -10).sqrt()
        assert bool((y == y[:, :1]).all())
        assert bool(((y[:, 0].double() / ref - 1).abs() <= 1.01 * 2.0 ** -24).all()), k
