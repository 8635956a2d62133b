"""What the linear attention's numbers are held to: inputs whose terms nearly cancel, so that a
context shows through its own rounding to bf16 what its operands were rounded to, and states whose
value is known to the last bit, or whose errors would add up over a sequence."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from linear_cases import inputs, oracle, wide
from mlx_omnia_amd.kernels import linear_attention
from mlx_omnia_amd.kernels.linear_attention import HipLinearAttention, LinearAttention, LinearBatch

pytestmark = pytest.mark.gpu

HALF, STEP = 2.0 ** -8, 2.0 ** -24   # half a step of bf16 and of fp32, relative
GEOMETRIES = [(2, 2, 128, 128), (4, 1, 128, 64), (3, 3, 128, 64), (4, 2, 64, 64), (2, 1, 64, 128), (3, 3, 64, 64)]


def layer(states, key_heads, scale=0.125):
    _, heads, key_dim, value_dim = states.shape
    mixer = LinearAttention(states, heads=heads, key_heads=key_heads, key_dim=key_dim, value_dim=value_dim, scale=scale,
                            dtype=torch.bfloat16)
    assert isinstance(mixer.strategy, HipLinearAttention)
    return mixer


def one_hot(tokens, heads, dim, where=0):
    rows = torch.zeros(tokens, heads, dim, dtype=torch.bfloat16, device="cuda")
    rows[:, :, where] = 1
    return rows


@pytest.mark.parametrize("heads,key_heads,key_dim,value_dim", GEOMETRIES)
@pytest.mark.parametrize("decay", [-0.5, -0.75, -3.0, -15.0, -30.0, -80.0])
def test_what_a_fast_decay_leaves(heads, key_heads, key_dim, value_dim, decay):
    """A token of no strength: the state is what the decay leaves of it, to 32 bits of itself and not
    of what it was."""
    states = 1 + torch.rand(1, heads, key_dim, value_dim, generator=torch.Generator().manual_seed(1)).cuda()
    want = states.double() * torch.exp(torch.tensor(decay, dtype=torch.float64))
    rows, v = one_hot(1, key_heads, key_dim, 3), torch.ones(1, heads, value_dim, dtype=torch.bfloat16, device="cuda")
    g = torch.full((1, heads), decay, device="cuda")
    out = layer(states, key_heads)(LinearBatch([0], [1]), rows, rows, v, g, torch.zeros(1, heads, device="cuda"))
    # An exponential to two steps of it, and a product (or the product and a sum).
    assert ((states.double() - want).abs() <= 6 * STEP * want).all()
    assert ((out.double() - 0.125 * want[:, :, 3]).abs() <= (HALF + 8 * STEP) * 0.125 * want[:, :, 3]).all()


@pytest.mark.parametrize("heads,key_heads,key_dim,value_dim", GEOMETRIES)
@pytest.mark.parametrize("fast,plus,minus", [(50, 51, 61), (20, 21, 31), (20, 25, 40), (40, 41, 50)])
def test_slow_decays_behind_fast_ones(heads, key_heads, key_dim, value_dim, fast, plus, minus):
    """Tokens at a log decay of -109, then slow ones: a later context is the difference of two
    weights, 1 - exp(-3e-4 n), which sums of decays in 32 bits (up to 2^-12 off here) would swallow."""
    n, g = 64, torch.full((64, heads), -3e-4, device="cuda")
    g[:fast] = -109.0
    v = torch.zeros(n, heads, value_dim, dtype=torch.bfloat16, device="cuda")
    v[plus], v[minus] = 1, -1
    states = torch.ones(1, heads, key_dim, value_dim, device="cuda")
    rows = one_hot(n, key_heads, key_dim)
    out = layer(states, key_heads)(LinearBatch([0], [n]), rows, rows, v, g).double()
    sums = torch.cumsum(g.double(), dim=0)
    first, second = torch.exp(sums[minus:] - sums[plus]), torch.exp(sums[minus:] - sums[minus])
    want = (0.125 * (first - second))[..., None]
    # One rounding of the result, and 2^-15 for each weight.
    allowed = HALF * want.abs() + 0.125 * 2 * 2.0 ** -15
    assert (want.abs() > 30 * allowed).any() and ((out[minus:] - want).abs() <= allowed).all()
    left = torch.exp(sums[-1] - sums[plus]) - torch.exp(sums[-1] - sums[minus])
    assert ((states[0, :, 0].double() - left[:, None]).abs() <= 16 * STEP).all()


def nearly_cancelling(n, seed=3):
    """Numbers of 24 bits in [1, 2), and others that are off by about 2^-12 of them, no two by the same."""
    gen = torch.Generator().manual_seed(seed)
    x = (1 + torch.rand(n, generator=gen)).float()
    return x.cuda(), (x * (1 + 2.0 ** -12 * (1 + torch.rand(n, generator=gen)))).float().cuda()


@pytest.mark.parametrize("tokens", [1, 20, 64, 130])
@pytest.mark.parametrize("heads,key_heads,key_dim,value_dim", GEOMETRIES)
def test_states_are_read_in_32_bits(heads, key_heads, key_dim, value_dim, tokens):
    """Contexts that are the difference of two rows of the state, which keys of zero leave as it is."""
    states = torch.zeros(1, heads, key_dim, value_dim, device="cuda")
    x, y = (t.view(heads, value_dim) for t in nearly_cancelling(heads * value_dim))
    i, j = 5, key_dim - 7
    states[0, :, i], states[0, :, j] = x, -y
    q = one_hot(tokens, key_heads, key_dim, i) + one_hot(tokens, key_heads, key_dim, j)
    v = torch.ones(tokens, heads, value_dim, dtype=torch.bfloat16, device="cuda")
    before = states.clone()
    out = layer(states, key_heads)(LinearBatch([0], [tokens]), q, torch.zeros_like(q), v, torch.zeros(tokens, heads, device="cuda"))
    want = 0.125 * (x.double() - y.double())
    # One rounding of the result; a few of the sum, of terms below 2 each.
    assert ((out.double() - want).abs() <= HALF * want.abs() + 0.125 * 8 * STEP * 2).all()
    assert torch.equal(states, before)


@pytest.mark.parametrize("first,second,last", [(0, 1, 64), (3, 40, 64), (33, 50, 60), (70, 71, 130), (0, 1, 5)])
@pytest.mark.parametrize("heads,key_heads,key_dim,value_dim", GEOMETRIES)
def test_weights_are_multiplied_in_32_bits(heads, key_heads, key_dim, value_dim, first, second, last):
    """Contexts that are the difference of two tokens' values, of nearly the same strength."""
    states = torch.zeros(1, heads, key_dim, value_dim, device="cuda")
    x, y = nearly_cancelling(heads)
    w = torch.zeros(last, heads, device="cuda")
    w[first], w[second] = x, y
    v = torch.zeros(last, heads, value_dim, dtype=torch.bfloat16, device="cuda")
    v[first], v[second] = 1, -1
    rows = one_hot(last, key_heads, key_dim, 9)
    out = layer(states, key_heads)(LinearBatch([0], [last]), rows, rows, v, torch.zeros(last, heads, device="cuda"), w)
    want = 0.125 * (x.double() - y.double())[:, None].expand(heads, value_dim)
    # One rounding of the result; a few of each weight's factors and of the sum, of terms below 2 each.
    allowed = HALF * want.abs() + 0.125 * 12 * STEP * 2
    assert ((out[second:].double() - want).abs() <= allowed).all()
    assert ((out[first:second].double() - 0.125 * x.double()[:, None]).abs() <= (HALF + 12 * STEP) * 0.125 * 2).all()
    assert not out[:first].any()


@pytest.mark.parametrize("chunks", [1 << 20, 2, 16])   # of a piece: uncut, many pieces, some
@pytest.mark.parametrize("decay", [-1e-4, -1.3e-5, -1e-3])
@pytest.mark.parametrize("heads,key_heads,key_dim,value_dim", [(2, 2, 128, 128), (2, 1, 128, 64), (1, 1, 64, 64)])
def test_slow_decays_over_a_long_sequence(monkeypatch, chunks, decay, heads, key_heads, key_dim, value_dim):
    """32,768 tokens of no strength and a fixed decay. What the rounding of each chunk's factor next to 1 would
    take away is the same for every chunk and number: the mean of all numbers' errors shows it, to
    which their own roundings, each its own, add little."""
    monkeypatch.setattr(linear_attention, "piece_chunks", lambda own, places: chunks)
    n = 32768
    gen = torch.Generator().manual_seed(2)
    states = 1 + torch.rand(1, heads, key_dim, value_dim, generator=gen).cuda()
    g = torch.full((n, heads), decay, device="cuda")
    want = states.double() * torch.exp(n * g[0, 0].double())
    rows, v = one_hot(n, key_heads, key_dim), torch.ones(n, heads, value_dim, dtype=torch.bfloat16, device="cuda")
    layer(states, key_heads)(LinearBatch([0], [n]), rows, rows, v, g, torch.zeros(n, heads, device="cuda"))
    off = (states.double() - want) / want
    # Each factor is off by two steps of what it takes away, or of itself (and its exponent's rounding), where it takes
    # more than half; one, of the state as it was, may be rounded next to 1. And 512 roundings of each number, of at most
    # a step of 2^-24, are off by 6 of their mean's deviations at most.
    mean = (5 * abs(decay) * n + 4) * STEP + 6 * (512 / states.numel()) ** 0.5 * STEP
    assert abs(off.mean().item()) <= mean
    assert off.abs().max().item() <= mean + 7 * 512 ** 0.5 * STEP


@pytest.mark.parametrize("tokens", [1, 4, 50, 64, 100])
@pytest.mark.parametrize("size", [1 << 20, 1])
@pytest.mark.parametrize("heads,key_heads,key_dim,value_dim", GEOMETRIES)
def test_states_keep_all_bits_of_what_is_added(monkeypatch, heads, key_heads, key_dim, value_dim, size, tokens):
    """A row of the state for each token (no more of them than rows): the token's value times its strength,
    in 32 bits, and nothing else."""
    monkeypatch.setattr(linear_attention, "piece_chunks", lambda own, places: size)
    n, gen = min(tokens, key_dim), torch.Generator().manual_seed(4)
    states = torch.zeros(1, heads, key_dim, value_dim, device="cuda")
    order = torch.randperm(key_dim, generator=gen)[:n]
    k = torch.zeros(n, key_heads, key_dim)
    k[torch.arange(n), :, order] = 1
    v = torch.randn(n, heads, value_dim, generator=gen).bfloat16().cuda()
    w = torch.rand(n, heads, generator=gen).cuda()
    k = k.bfloat16().cuda()
    layer(states, key_heads)(LinearBatch([0], [n]), k, k, v, torch.zeros(n, heads, device="cuda"), w)
    want = torch.zeros_like(states)
    want[0, :, order.cuda()] = (v.float() * w[..., None]).transpose(0, 1)
    assert torch.equal(states, want)


@pytest.mark.parametrize("size", [1 << 20, 4])
@pytest.mark.parametrize("tokens", [200, 1500])
@pytest.mark.parametrize("heads,key_heads,key_dim,value_dim", GEOMETRIES[:4])
def test_states_of_prompts_as_a_whole(monkeypatch, heads, key_heads, key_dim, value_dim, tokens, size):
    """The states' error as a whole (2-norm). A chunk rounds a state at most 12 times in its products
    and three times in its decay and its pieces, by at most a step of 2^-24 of what it comes to, one
    way or the other: the square root of their number together. (Values in two parts, of 16 bits, would
    be off by 2^-18.)"""
    monkeypatch.setattr(linear_attention, "piece_chunks", lambda own, places: size)
    made, _, states, slots = inputs([tokens], heads, key_heads, key_dim, value_dim, device="cuda", strengths=True)
    before = wide(states)
    layer(states, key_heads)(LinearBatch(slots, [tokens]), **made)
    _, left, _, _ = oracle(*(wide(made[name]) for name in ("queries", "keys", "values", "log_decay", "strengths")), before,
                           slots, [tokens], 0.125)
    off = np.linalg.norm(wide(states)[slots[0]] - left[slots[0]]) / np.linalg.norm(left[slots[0]])
    print(f"states off by {off:.3g}", flush=True)
    assert off <= (15 * -(-tokens // 64)) ** 0.5 * STEP
