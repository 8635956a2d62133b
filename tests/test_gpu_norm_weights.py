"""The gated norm and the join of two blocks with weights that are views of packed parameters: a
kernel that cannot read them leaves the call to the Core chain."""

from __future__ import annotations

import pytest
import torch

from mlx_omnia_amd.kernels.block_norm import BlockNorm, DefaultBlockNorm, HipBlockNorm
from mlx_omnia_amd.kernels.gated_norm import DefaultGatedRmsNorm, GatedRmsNorm, HipGatedRmsNorm
from mlx_omnia_amd.kernels.leaf import RMSNormLeaf
from norm_cases import EPS, block_case, check_block, check_gated, gated_case

pytestmark = pytest.mark.gpu


def odd(weight):
    """The same values a bf16 number past an aligned address."""
    return torch.cat([weight.new_zeros(1), weight])[1:]


def strided(weight):
    """The same values as a column of a matrix."""
    return torch.stack([weight, torch.zeros_like(weight)], dim=1)[:, 0]


def aligned(weight):
    """The same values in the middle of a packed parameter, 16 bytes or more from its start."""
    return torch.cat([weight.new_zeros(8), weight, weight])[8 : 8 + weight.numel()]


@pytest.mark.parametrize("view,served", [(odd, False), (strided, False), (aligned, True)])
@pytest.mark.parametrize("whole", [False, True])
def test_gated_norm(view, served, whole):
    x, gate, weight = gated_case(5, 256, 256 if whole else 64, device="cuda")
    weight = view(weight)
    norm = GatedRmsNorm(RMSNormLeaf(weight, EPS), group=64)
    assert isinstance(norm.strategy, HipGatedRmsNorm if served else DefaultGatedRmsNorm)
    check_gated(norm(x, gate), x, gate, weight, 64, "silu", False)
    weight.mul_(0.5)   # what is written to the parameter counts
    check_gated(norm(x, gate), x, gate, weight, 64, "silu", False)


@pytest.mark.parametrize("view,served", [(odd, False), (strided, False), (aligned, True)])
@pytest.mark.parametrize("which", ["pre", "post", "both"])
def test_block_norm(view, served, which):
    x, block, _, pre, post = block_case(5, 256, None, True, device="cuda")
    pre, post = view(pre) if which != "post" else pre, view(post) if which != "pre" else post
    join = BlockNorm(RMSNormLeaf(pre, EPS), RMSNormLeaf(post, 1e-5), residual_scale=0.5, block_scale=1.5)
    assert isinstance(join.strategy, HipBlockNorm if served else DefaultBlockNorm)
    check_block(join(x, block), x, block, None, pre, post, None, 0.5, 1.5)
    pre.mul_(0.5), post.mul_(2.0)
    check_block(join(x, block), x, block, None, pre, post, None, 0.5, 1.5)
