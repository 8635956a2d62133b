"""HIP gated norm and join of two blocks against the float64 oracle: every width of lanes and waves,
groups and rows that do not fill them, strides, gates at the edge, and refusals."""

from __future__ import annotations

import math

import pytest
import torch

from mlx_omnia_amd.kernels.block_norm import BlockNorm, HipBlockNorm
from mlx_omnia_amd.kernels.gated_norm import GatedRmsNorm, HipGatedRmsNorm
from mlx_omnia_amd.kernels.leaf import RMSNormLeaf
from norm_cases import block_case, check_block, check_gated, gated_case

pytestmark = pytest.mark.gpu

GROUPS = [8, 24, 64, 72, 128, 136, 256, 264, 512, 520, 1024, 1032, 2048, 2560, 4096, 5000, 8192]


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("gate_first", [False, True])
def test_gated_groups(group, gate_first):
    for rows, groups, act in ((1, 1, "silu"), (5, 3, "sigmoid"), (33, 2, "silu")):
        print(f"gated_rms_norm rows={rows} groups={groups} of {group} {act} {gate_first}", flush=True)
        x, gate, weight = gated_case(rows, group * groups, group if rows != 33 else group * groups, device="cuda")
        norm = GatedRmsNorm(RMSNormLeaf(weight), group=group, activation=act, gate_first=gate_first)
        assert isinstance(norm.strategy, HipGatedRmsNorm)
        check_gated(norm(x, gate), x, gate, weight, group, act, gate_first)


@pytest.mark.parametrize("rows", [1, 2, 700, 5000])
def test_gated_rows(rows):
    x, gate, weight = gated_case(rows, 1024, 128, device="cuda")
    norm = GatedRmsNorm(RMSNormLeaf(weight), group=128)
    check_gated(norm(x, gate), x, gate, weight, 128, "silu", False)
    heads = norm(x.unflatten(1, (8, 128)), gate.unflatten(1, (8, 128)))
    assert heads.shape == (rows, 8, 128) and torch.equal(heads.flatten(1), norm(x, gate))


def test_gated_views():
    """Slices of wider rows, heads of them, unaligned and transposed rows: as their copies."""
    x, gate, weight = gated_case(40, 512, 64, device="cuda")
    norm = GatedRmsNorm(RMSNormLeaf(weight), group=64)
    want = norm(x, gate)
    rows = torch.cat([gate, x, gate], dim=1)
    assert torch.equal(norm(rows[:, 512:1024], rows[:, :512]), want)
    heads = rows.unflatten(1, (24, 64))
    assert torch.equal(norm(heads[:, 8:16], heads[:, :8]).flatten(1), want)
    odd = torch.cat([x.new_zeros(1), x.flatten()])[1:].view(x.shape)
    assert torch.equal(norm(odd, gate), want)
    assert torch.equal(norm(x.t().contiguous().t(), gate), want)
    assert torch.equal(norm(x.view(8, 5, 512), gate.view(8, 5, 512)).view(40, 512), want)
    assert norm(x[:0], gate[:0]).shape == (0, 512)


@pytest.mark.parametrize("gate_first", [False, True])
def test_gated_edges(gate_first):
    x, gate, weight = gated_case(8, 128, 128, device="cuda")
    x[0], x[1] = 0.0, 1e18
    gate[2], gate[3], gate[4] = 300.0, -300.0, 0.0
    x[5, 3] = math.nan
    norm = GatedRmsNorm(RMSNormLeaf(weight), gate_first=gate_first)
    out = norm(x, gate)
    fine = [0, 1, 2, 3, 4, 6, 7]
    assert torch.isfinite(out[fine]).all()
    check_gated(out[fine], x[fine], gate[fine], weight, 128, "silu", gate_first)
    assert out[5].isnan().all()


@pytest.mark.parametrize("gate_first", [False, True])
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
def test_gated_at_the_ends_of_the_range(gate_first, act):
    """Values and gates whose product is out of fp32's range where no step of the formula is."""
    x, gate, weight = gated_case(6, 128, 128, device="cuda")
    x[0] *= 1e15
    gate[0, ::2] = -1e30          # times a sigmoid of zero
    x[1] *= 1e-15
    gate[1] = gate[1] * 1e-30
    if not gate_first:            # (the norm of such products has no fp32 square)
        x[2] *= 1e15
        gate[2] = gate[2].abs() * 1e25
    x[3, 5], gate[3, 5] = 2e18, -3e38
    norm = GatedRmsNorm(RMSNormLeaf(weight), activation=act, gate_first=gate_first)
    out = norm(x, gate)
    assert torch.isfinite(out).all()
    check_gated(out, x, gate, weight, 128, act, gate_first)


HIDDENS = [8, 64, 504, 512, 520, 1024, 1032, 2048, 2560, 4096, 4104, 5120, 8192, 8200, 16384]


@pytest.mark.parametrize("hidden", HIDDENS)
@pytest.mark.parametrize("gate,act,post", [(None, None, False), (None, None, True), ("rows", "sigmoid", True),
                                           ("row", None, True), ("rows", None, False)])
def test_block_widths(hidden, gate, act, post):
    for rows in (1, 3):
        print(f"block_norm rows={rows} hidden={hidden} {gate} {act} {post}", flush=True)
        x, block, g, pre, behind = block_case(rows, hidden, gate, post, device="cuda")
        join = BlockNorm(RMSNormLeaf(pre), None if behind is None else RMSNormLeaf(behind, 1e-5), residual_scale=0.75,
                         block_scale=1.5, activation=act)
        assert isinstance(join.strategy, HipBlockNorm)
        check_block(join(x, block, g), x, block, g, pre, behind, act, 0.75, 1.5)


@pytest.mark.parametrize("rows", [2, 300, 5000])
@pytest.mark.parametrize("hidden", [1000, 2560])
def test_block_rows(rows, hidden):
    x, block, g, pre, behind = block_case(rows, hidden, "rows", True, device="cuda")
    join = BlockNorm(RMSNormLeaf(pre), RMSNormLeaf(behind, 1e-5), residual_scale=3.5, block_scale=0.5, activation="sigmoid")
    check_block(join(x, block, g), x, block, g, pre, behind, "sigmoid", 3.5, 0.5)


def test_block_views():
    x, block, g, pre, behind = block_case(12, 256, "rows", True, device="cuda")
    join = BlockNorm(RMSNormLeaf(pre), RMSNormLeaf(behind), activation="sigmoid")
    want = join(x, block, g)
    wide = torch.cat([x, block, g], dim=1)
    for got in (join(wide[:, :256], wide[:, 256:512], wide[:, 512:]), join(x.t().contiguous().t(), block, g),
                [t.view(12, 256) for t in join(*(t.view(3, 4, 256) for t in (x, block, g)))]):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = join(x, block, g[0])
    assert all(torch.equal(a, b) for a, b in zip(one, join(x, block, g[:1].expand(12, 256))))
    assert [t.shape for t in join(x[:0], block[:0], g[:0])] == [(0, 256), (0, 256)]
    assert torch.equal(join(x[0], block[0], g[0])[1], want[1][0])


def test_captured_and_replayed():
    x, block, g, pre, behind = block_case(300, 2560, "rows", True, device="cuda")
    join = BlockNorm(RMSNormLeaf(pre), RMSNormLeaf(behind), activation="sigmoid")
    norm = GatedRmsNorm(RMSNormLeaf(behind), group=2560)
    join(x, block, g), norm(x, g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = (*join(x, block, g), norm(x, g))
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        want = (*join(x, block, g), norm(x, g))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_the_operators_for_compilers_equal_their_calls():
    import mlx_omnia_amd.runtime.torch_ops  # noqa: F401

    x, block, g, pre, behind = block_case(30, 512, "rows", True, device="cuda")
    join = BlockNorm(RMSNormLeaf(pre, 1e-6), RMSNormLeaf(behind, 1e-5), residual_scale=0.5, block_scale=1.5, activation="sigmoid")
    norm = GatedRmsNorm(RMSNormLeaf(behind, 1e-6), group=64)

    def chain(x, block, g):
        s, n = torch.ops.omnia.block_norm(x, block, pre, behind, g, 1e-6, 1e-5, 0.5, 1.5, True)
        return s, n, torch.ops.omnia.gated_rms_norm(n, g, behind, 64, 1e-6)

    s, n = join(x, block, g)
    want = s, n, norm(n, g)
    assert all(torch.equal(a, b) for a, b in zip(chain(x, block, g), want))
    compiled = torch.compile(chain, fullgraph=True, backend="aot_eager")
    assert all(torch.equal(a, b) for a, b in zip(compiled(x, block, g), want))


def test_refusals_and_hand_offs():
    x, block, g, pre, behind = block_case(4, 64, "rows", True, device="cuda")
    join, norm = BlockNorm(RMSNormLeaf(pre)), GatedRmsNorm(RMSNormLeaf(pre))
    with pytest.raises(ValueError):
        join(x, block.cpu())
    with pytest.raises(ValueError):
        norm(x, g.cpu())
    assert join(x.float(), block.float())[0].dtype == torch.float32
    leaf = x.clone().requires_grad_()
    join(leaf, block)[1].float().sum().backward()
    norm(leaf, g).float().sum().backward()
    assert torch.isfinite(leaf.grad).all()
