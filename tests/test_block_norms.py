"""The gated norm and the join of two blocks on the CPU: the Core chains against the float64
oracle, their gradients, and what they refuse."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mlx_omnia_amd.kernels.block_norm import BlockNorm, DefaultBlockNorm
from mlx_omnia_amd.kernels.block_norm import applies as block_applies
from mlx_omnia_amd.kernels.gated_norm import DefaultGatedRmsNorm, GatedRmsNorm
from mlx_omnia_amd.kernels.gated_norm import applies as gated_applies
from mlx_omnia_amd.kernels.leaf import RMSNormLeaf
from norm_cases import block_case, check_block, check_gated, gated_case


@pytest.mark.parametrize("rows,width,group", [(3, 64, 64), (2, 96, 24), (1, 512, 128), (0, 64, 64)])
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("gate_first", [False, True])
@pytest.mark.parametrize("whole", [False, True])
def test_gated_core_against_the_oracle(rows, width, group, act, gate_first, whole):
    x, gate, weight = gated_case(rows, width, width if whole else group)
    norm = GatedRmsNorm(RMSNormLeaf(weight), group=group, activation=act, gate_first=gate_first)
    assert isinstance(norm.strategy, DefaultGatedRmsNorm)
    check_gated(norm(x, gate), x, gate, weight, group, act, gate_first)


def test_gated_core_of_heads():
    x, gate, weight = gated_case(3, 64, 16)
    norm = GatedRmsNorm(RMSNormLeaf(weight))
    out = norm(x.unflatten(1, (4, 16)), gate.unflatten(1, (4, 16)))
    assert out.shape == (3, 4, 16)
    check_gated(out.flatten(1), x, gate, weight, 16, "silu", False)


@pytest.mark.parametrize("rows,hidden", [(1, 64), (3, 40), (0, 16)])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [None, "rows", "row"])
@pytest.mark.parametrize("act", [None, "sigmoid"])
def test_block_core_against_the_oracle(rows, hidden, post, gate, act):
    x, block, g, pre, behind = block_case(rows, hidden, gate, post)
    join = BlockNorm(RMSNormLeaf(pre), None if behind is None else RMSNormLeaf(behind, 1e-5), residual_scale=0.75,
                     block_scale=1.5, activation=act)
    assert isinstance(join.strategy, DefaultBlockNorm)
    check_block(join(x, block, g), x, block, g, pre, behind, act, 0.75, 1.5)


def test_gradients_against_differences():
    gen = torch.Generator().manual_seed(1)
    x, gate, block = (torch.randn(2, 16, generator=gen, dtype=torch.float64, requires_grad=True) for _ in range(3))
    weight = torch.randn(8, generator=gen, dtype=torch.float64)
    for first in (False, True):
        norm = GatedRmsNorm(RMSNormLeaf(weight), gate_first=first)
        assert torch.autograd.gradcheck(norm, (x, gate))
    join = BlockNorm(RMSNormLeaf(weight.repeat(2)), RMSNormLeaf(weight.repeat(2)), residual_scale=0.5, block_scale=2.0,
                     activation="sigmoid")
    assert torch.autograd.gradcheck(join, (x, block, gate))


def test_refusals():
    w = torch.ones(64)
    for kwargs in (dict(group=48), dict(activation="gelu"), dict(group=0)):
        with pytest.raises(ValueError):
            GatedRmsNorm(RMSNormLeaf(w), **kwargs)
    with pytest.raises(ValueError):
        GatedRmsNorm(RMSNormLeaf(torch.ones(2, 32)))
    norm = GatedRmsNorm(RMSNormLeaf(w), group=32)
    for x, gate in ((torch.ones(2, 64), torch.ones(2, 32)), (torch.ones(2, 96), torch.ones(2, 96)),
                    (torch.ones(2, 32), torch.ones(2, 32))):
        with pytest.raises(ValueError):
            norm(x, gate)
    with pytest.raises(ValueError):
        BlockNorm(RMSNormLeaf(w), RMSNormLeaf(torch.ones(32)))
    with pytest.raises(ValueError):
        BlockNorm(RMSNormLeaf(w), activation="tanh")
    join = BlockNorm(RMSNormLeaf(w))
    x = torch.ones(2, 64)
    for args in ((x, x[:1]), (x[:, :32], x[:, :32]), (x, x, torch.ones(2, 1)), (x, x, torch.ones(1, 64))):
        with pytest.raises(ValueError):
            join(*args)
    assert np.array_equal([gated_applies(n) for n in (8, 8192, 4, 8200, 0)], [True, True, False, False, False])
    assert np.array_equal([block_applies(n) for n in (8, 16384, 12, 16392, 0)], [True, True, False, False, False])


def test_the_operators_for_compilers_give_shapes_without_a_device():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from mlx_omnia_amd.runtime import torch_ops

    assert {"gated_rms_norm", "block_norm"} <= set(torch_ops.REGISTERED)
    with FakeTensorMode():
        x, w = torch.empty(3, 5, 64, dtype=torch.bfloat16), torch.empty(64, dtype=torch.bfloat16)
        y = torch.ops.omnia.gated_rms_norm(x.transpose(0, 1), x.transpose(0, 1), w, 64, 1e-6)
        assert y.shape == (5, 3, 64) and y.dtype == torch.bfloat16 and y.is_contiguous()
        s, n = torch.ops.omnia.block_norm(x, x, w, None, None, 1e-6, 0.0, 1.0, 1.0, False)
        assert s.shape == n.shape == x.shape and n.dtype == torch.bfloat16
