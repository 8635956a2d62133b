"""The sums of squares behind the gated norm and the join of two blocks: rows whose squares are one
of about 1 and thousands of just under half a step of it, which sums that add them to it one by one
lose one by one."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mlx_omnia_amd.kernels.block_norm import BlockNorm, HipBlockNorm
from mlx_omnia_amd.kernels.gated_norm import GatedRmsNorm, HipGatedRmsNorm
from mlx_omnia_amd.kernels.leaf import RMSNormLeaf
from norm_cases import EPS, _wide, oracle

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24
# Of a result, relative: a sum of at most 16 squares in turn, a tree of 8 x 64 and 8 waves' in turn, under 40
# roundings halved by the root, and those of the mean, the root, the reciprocal and three products.
NEAR = 28 * STEP


def rows_of(count, width):
    """A large value first in a lane's share, another one in each row, and small ones behind it."""
    gen = torch.Generator().manual_seed(width)
    large = (1 + torch.arange(count) % 52 / 128).double()                   # squares in [1, 2)
    small = torch.full((count, width), (0.47 * 2.0 ** -23) ** 0.5).bfloat16()
    assert 2.0 ** -26 < small.double().max() ** 2 < 2.0 ** -24
    at = torch.randint(0, 64, (count,), generator=gen) * 8 % width
    small[torch.arange(count), at] = large.bfloat16()
    return small.cuda(), (1 + torch.randint(0, 128, (width,), generator=gen) / 128).bfloat16().cuda()


def check(got, want):
    """Results that are not so near the middle between two bf16 numbers that their errors may round
    them otherwise are the nearest one."""
    got = _wide(got)
    size, exponent = np.frexp(np.abs(want))
    steps = size * 2.0 ** 8
    sure = np.abs(steps - np.floor(steps) - 0.5) > NEAR * steps
    nearest = np.copysign(np.ldexp(np.round(steps), exponent - 8), want)
    assert sure.mean() > 0.99 and np.array_equal(got[sure], nearest[sure])


@pytest.mark.parametrize("group", [64, 512, 1024, 2048, 4096, 8192])
def test_gated_norm(group):
    x, weight = rows_of(104, group)
    norm = GatedRmsNorm(RMSNormLeaf(weight, EPS), activation="sigmoid")
    assert isinstance(norm.strategy, HipGatedRmsNorm)
    gate = torch.full_like(x, 40.0)   # a sigmoid of 1
    check(norm(x, gate), oracle.gated_rms_norm(_wide(x), _wide(gate), _wide(weight), group, EPS, False, False))


@pytest.mark.parametrize("hidden", [512, 2048, 8192, 16384])
def test_block_norm(hidden):
    x, weight = rows_of(104, hidden)
    join = BlockNorm(RMSNormLeaf(weight, EPS))
    assert isinstance(join.strategy, HipBlockNorm)
    check(join(x, torch.zeros_like(x))[1], oracle.block_norm(_wide(x), np.zeros(x.shape), _wide(weight), EPS)[1])
