"""Linear attention on the CPU: the Core chain against the float64 oracle, its gradients, and what
batches and layers refuse."""

from __future__ import annotations

import math

import pytest
import torch

from linear_cases import check, inputs
from mlx_omnia_amd.kernels.linear_attention import (DefaultLinearAttention, LinearAttention, LinearBatch, applies,
                                                    piece_chunks)


def layer(states, key_heads, decay=None, **more):
    _, heads, key_dim, value_dim = states.shape
    return LinearAttention(states, heads=heads, key_heads=key_heads, key_dim=key_dim, value_dim=value_dim,
                           scale=key_dim ** -0.5, dtype=torch.bfloat16, decay=decay, **more)


@pytest.mark.parametrize("tokens", [[1], [1, 1, 1], [5, 0, 1, 70], [64], [65, 129]])
@pytest.mark.parametrize("decay,strengths", [("token", False), ("token", True), ("head", False)])
def test_core_against_the_oracle(tokens, decay, strengths):
    made, fixed, states, slots = inputs(tokens, 4, 2, 16, 8, seed=len(tokens), strengths=strengths, decay=decay)
    before = states.clone()
    mixer = layer(states, 2, fixed)
    assert isinstance(mixer.strategy, DefaultLinearAttention)
    out = mixer(LinearBatch(slots, tokens, device="cpu"), **made)
    assert out.dtype == torch.bfloat16 and out.shape == made["values"].shape
    check(out, states, made, fixed, before, slots, tokens, 0.25)
    rest = [s for s in range(len(states)) if s not in slots or tokens[slots.index(s)] == 0]
    assert torch.equal(states[rest], before[rest])


def test_core_in_two_calls_as_in_one():
    made, _, states, slots = inputs([100], 4, 2, 16, 8, dtype=torch.float64)
    made["log_decay"] = made["log_decay"].double()
    whole, parts = states.double(), states.double()
    one = layer(whole, 2)(LinearBatch(slots, [100], device="cpu"), **made)
    cut = [layer(parts, 2)(LinearBatch(slots, [n], device="cpu"),
                           **{k: None if t is None else t[a : a + n] for k, t in made.items()})
           for a, n in ((0, 37), (37, 1), (38, 62))]
    torch.testing.assert_close(torch.cat(cut), one, rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(parts, whole, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_core_keeps_what_is_not_finite_from_earlier_tokens(bad):
    made, _, states, slots = inputs([70], 2, 2, 16, 8)
    made["values"] = made["values"].clone()
    made["values"][40, 1, 3] = bad
    before = states.clone()
    out = layer(states, 2)(LinearBatch(slots, [70], device="cpu"), **made)
    assert torch.isfinite(out[:40]).all() and not torch.isfinite(out[40:, 1, 3]).any()
    check(out, states, made, None, before, slots, [70], 0.25)


def test_core_forgets_all():
    """A log decay of -inf leaves nothing of what was before, even of an infinity's own -inf differences."""
    made, _, states, slots = inputs([9], 2, 1, 16, 8)
    made["log_decay"][3] = -math.inf
    made["log_decay"][4] = -1e30
    before = states.clone()
    out = layer(states, 1)(LinearBatch(slots, [9], device="cpu"), **made)
    assert torch.isfinite(out).all()
    check(out, states, made, None, before, slots, [9], 0.25)


def test_core_gradients_against_differences():
    """Central differences in float64: the truncation of steps of 1e-6 and the rounding of sums of a
    hundred terms stay below 1e-6 of gradients of about one."""
    made, _, states, slots = inputs([5, 2], 4, 2, 8, 4, strengths=True, dtype=torch.float64)
    leaves = {k: t.detach().double().requires_grad_() for k, t in made.items()}
    batch = LinearBatch(slots, [5, 2], device="cpu")

    def run(*tensors):
        pool = states.double()   # each call its own pool: the call moves it on
        return layer(pool, 2)(batch, **dict(zip(leaves, tensors)))

    assert torch.autograd.gradcheck(run, tuple(leaves.values()), eps=1e-6, atol=1e-6, rtol=1e-6)


def test_a_batch_refuses():
    for slots, tokens in (([0, 0], [1, 1]), ([0], [1, 2]), ([-1], [1]), ([0], [-1]), ([0], [1 << 24])):
        with pytest.raises(ValueError):
            LinearBatch(slots, tokens, device="cpu")


def test_lists_cover_every_token_once():
    """Whatever the lengths and heads: each token in one step or piece, pieces of a sequence in order,
    of whole chunks but the last, and their places one behind the other."""
    gen = torch.Generator().manual_seed(3)
    for trial in range(60):
        count = int(torch.randint(0, 12, (1,), generator=gen))
        tokens = [int(2 ** (14 * float(torch.rand(1, generator=gen)))) - 1 for _ in range(count)]
        slots = torch.randperm(count + 3, generator=gen).tolist()[:count]
        heads = (1, 4, 32, 64)[trial % 4]
        batch, places = LinearBatch(slots, tokens, device="cpu"), (256, 512, 1024)[trial % 3]
        lists = batch.lists(heads, places)
        assert lists is batch.lists(heads, places)
        seen, places = torch.zeros(batch.total, dtype=torch.int64), []
        for slot, first, n in lists.steps.tolist():
            assert tokens[slots.index(slot)] == n
            seen[first : first + n] += 1
        by_slot: dict = {}
        for i, (slot, first, n, place, kind) in enumerate(lists.runs.tolist()):
            seen[first : first + n] += 1
            assert (kind & 2 == 0) == (i < lists.handed_on) and n > 0
            by_slot.setdefault(slot, []).append((first, n, place, kind))
        for slot, runs in by_slot.items():
            runs.sort()
            assert sum(n for _, n, _, _ in runs) == tokens[slots.index(slot)]
            assert [kind for *_, kind in runs] == [(i == 0) + 2 * (i == len(runs) - 1) for i in range(len(runs))]
            assert all(n % 64 == 0 for _, n, _, _ in runs[:-1])
            if len(runs) == 1:
                assert runs[0][2] == -1
            else:
                assert [p for _, _, p, _ in runs] == list(range(runs[0][2], runs[0][2] + len(runs)))
                places += [p for _, _, p, _ in runs]
        assert (seen == 1).all() and sorted(places) == list(range(lists.pieces))
        assert sorted(lists.chains.tolist()) == sorted(
            [runs[0][2], len(runs)] for runs in by_slot.values() if len(runs) > 2)
    empty = LinearBatch([], [], device="cpu")
    assert empty.total == 0 and empty.lists(4, 512).steps.shape == (0, 3) and empty.lists(4, 512).runs.shape == (0, 5)
    assert LinearBatch([4, 2, 9], [3, 0, 2], device="cpu").lists(4, 512).steps.tolist() == [[4, 0, 3], [9, 3, 2]]


def test_a_layer_refuses():
    states = torch.zeros(2, 4, 16, 8)
    for kwargs in (dict(heads=4, key_heads=3), dict(heads=4, key_heads=0), dict(heads=5, key_heads=1)):
        with pytest.raises(ValueError):
            LinearAttention(states, key_dim=16, value_dim=8, scale=1.0, dtype=torch.bfloat16, **kwargs)
    with pytest.raises(ValueError):
        LinearAttention(states.bfloat16(), heads=4, key_heads=2, key_dim=16, value_dim=8, scale=1.0, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        layer(states, 2, torch.zeros(3))
    made, _, pool, slots = inputs([3], 4, 2, 16, 8, slots=2)
    mixer, batch = layer(pool, 2), LinearBatch(slots, [3], device="cpu")
    for change in (dict(queries=made["queries"][:2]), dict(keys=made["keys"][:, :1]), dict(values=made["values"][..., :4]),
                   dict(log_decay=None), dict(log_decay=made["log_decay"][:, :2]), dict(strengths=torch.ones(3))):
        with pytest.raises(ValueError):
            mixer(batch, **{**made, **change})
    with pytest.raises(ValueError):
        mixer(LinearBatch([2], [3], device="cpu"), **made)


def test_an_empty_call():
    made, _, states, _ = inputs([], 4, 2, 16, 8, slots=2)
    assert layer(states, 2)(LinearBatch([], [], device="cpu"), **made).shape == (0, 4, 8)
    made, _, states, slots = inputs([0], 4, 2, 16, 8, slots=2)
    before = states.clone()
    assert layer(states, 2)(LinearBatch(slots, [0], device="cpu"), **made).shape == (0, 4, 8)
    assert torch.equal(states, before)


def test_which_geometries_the_kernels_take():
    assert applies(32, 16, 128, 128) and applies(64, 1, 128, 64) and applies(6, 2, 64, 128)
    assert not applies(32, 16, 96, 128) and not applies(32, 16, 128, 256) and not applies(5, 2, 64, 64)
    assert not applies(0, 1, 64, 64) and not applies(8192, 1, 64, 64)


def test_a_pool_that_is_a_parameter_is_moved_on_without_gradients():
    made, _, states, slots = inputs([70], 2, 1, 16, 8, slots=1)
    clean, pool = states.clone(), torch.nn.Parameter(states.clone())
    want = layer(clean, 1)(LinearBatch(slots, [70], device="cpu"), **made)
    leaf = made["values"].clone().requires_grad_()
    out = layer(pool, 1)(LinearBatch(slots, [70], device="cpu"), **{**made, "values": leaf})
    assert torch.equal(out, want) and torch.equal(pool.detach(), clean)
    out.float().sum().backward()
    assert pool.grad is None and torch.isfinite(leaf.grad).all()


def test_pieces_for_the_least_time():
    assert piece_chunks([], 4) == 1 and piece_chunks([5], 1) == 5 and piece_chunks([1] * 40, 16) == 1
    assert piece_chunks([512], 16) == 32            # as many pieces as places
    assert piece_chunks([64] * 16, 16) == 64        # all places taken: whole
    for chunks, places in (([24, 13, 2, 14, 1], 16), ([300, 1, 1], 8), ([7] * 50, 4)):
        assert 1 <= piece_chunks(chunks, places) <= max(chunks)
