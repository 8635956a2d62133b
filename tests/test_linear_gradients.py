"""The Core chain of the linear attention: gradients across its chunks, of a layer's fixed decay and behind
values that are not finite; and pools of more than 32 bits."""

from __future__ import annotations

import math

import pytest
import torch

from linear_cases import inputs, oracle, wide
from mlx_omnia_amd.kernels.linear_attention import CHUNK, LinearAttention, LinearBatch


def layer(states, key_heads, decay=None):
    _, heads, key_dim, value_dim = states.shape
    return LinearAttention(states, heads=heads, key_heads=key_heads, key_dim=key_dim, value_dim=value_dim, scale=0.5,
                           dtype=torch.bfloat16, decay=decay)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_pool_of_64_bits_is_kept_in_64(dtype):
    made, _, states, slots = inputs([70, 1], 4, 2, 16, 8, strengths=True, dtype=dtype)
    pool = states.double() + 2.0 ** -40 * torch.rand(states.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    before = pool.clone()
    batch = LinearBatch(slots, [70, 1], device="cpu")
    zero = {**made, "values": torch.zeros_like(made["values"]), "log_decay": torch.zeros_like(made["log_decay"])}
    layer(pool, 2)(batch, **zero)
    assert torch.equal(pool, before)
    out = layer(pool, 2)(batch, **made)
    assert out.dtype == dtype
    _, left, _, sizes = oracle(*(wide(made[name]) for name in ("queries", "keys", "values", "log_decay", "strengths")),
                               wide(before), slots, [70, 1], 0.5)
    # Under 500 roundings of 2^-53 each.
    assert (abs(wide(pool) - left) <= 500 * 2.0 ** -53 * sizes).all()


def check_gradients(run, leaves):
    """Central differences in float64: the truncation of steps of 1e-6 and the rounding of sums of a thousand
    terms stay below 1e-6 of gradients of about one."""
    assert torch.autograd.gradcheck(run, tuple(leaves), eps=1e-6, atol=1e-6, rtol=1e-6)


def test_gradients_across_chunks():
    """A sequence that ends in its second chunk: what earlier tokens add reaches it through the state."""
    tokens = [CHUNK + 3, 1]
    made, _, states, slots = inputs(tokens, 2, 1, 3, 2, strengths=True, dtype=torch.float64)
    made["log_decay"] = made["log_decay"] * 0.05   # of which enough is left after a chunk
    leaves = {name: t.detach().double().requires_grad_() for name, t in made.items()}
    batch = LinearBatch(slots, tokens, device="cpu")
    run = lambda *tensors: layer(states.double(), 1)(batch, **dict(zip(leaves, tensors)))  # noqa: E731
    check_gradients(run, leaves.values())
    out = run(*leaves.values())
    first = torch.autograd.grad(out[CHUNK + 2].sum(), [leaves[name] for name in ("keys", "values", "log_decay", "strengths")])
    assert all((g[:CHUNK].abs() > 1e-6).any() for g in first)


def test_gradients_of_a_fixed_decay():
    tokens = [CHUNK + 2, 3]
    made, fixed, states, slots = inputs(tokens, 2, 2, 2, 2, decay="head", dtype=torch.float64)
    leaves = [made[name].detach().double().requires_grad_() for name in ("queries", "keys", "values")]
    decay = (fixed.double() * 0.2).requires_grad_()
    batch = LinearBatch(slots, tokens, device="cpu")
    check_gradients(lambda q, k, v, g: layer(states.double(), 2, g)(batch, q, k, v), [*leaves, decay])


def test_gradients_a_token_at_a_time():
    """Beside a value that is not finite the chain takes one token after another: the gradients of earlier tokens
    from contexts that do not see it are those of a call without it. (Its own and later tokens' are autograd's
    zeros times an infinity.)"""
    n, at = 12, 7
    made, _, states, slots = inputs([n], 2, 1, 3, 4, strengths=True, dtype=torch.float64)
    batch, grads = LinearBatch(slots, [n], device="cpu"), []
    for bad in (False, True):
        leaves = {name: t.detach().double().requires_grad_() for name, t in made.items()}
        values = leaves["values"]
        if bad:
            values = values.clone()
            values[at, 1, 2] = math.inf
        out = layer(states.double(), 1)(batch, **{**leaves, "values": values})
        assert torch.isfinite(out[:at]).all() and torch.isfinite(out[at:, 1, 2]).all() != bad
        grads.append(torch.autograd.grad(out[:at].square().sum(), list(leaves.values())))
    for without, beside in zip(*grads):
        torch.testing.assert_close(beside[:at], without[:at], rtol=1e-12, atol=1e-12)


def test_gradients_of_the_norms_weights():
    from mlx_omnia_amd.kernels.block_norm import BlockNorm
    from mlx_omnia_amd.kernels.gated_norm import GatedRmsNorm
    from mlx_omnia_amd.kernels.leaf import RMSNormLeaf

    gen = torch.Generator().manual_seed(6)
    x, gate, block, pre, post = (torch.randn(shape, generator=gen, dtype=torch.float64, requires_grad=True)
                                 for shape in ((3, 16), (3, 16), (3, 16), (16,), (16,)))
    narrow = torch.randn(8, generator=gen, dtype=torch.float64, requires_grad=True)
    for first in (False, True):
        for weight in (narrow, pre):   # of each group, and of the row
            check_gradients(lambda x, gate, w: GatedRmsNorm(RMSNormLeaf(w), group=8, gate_first=first)(x, gate),
                            [x, gate, weight])
    for g in (gate, post.detach().clone().requires_grad_()):   # a gate of each row, and one for all
        check_gradients(lambda x, block, g, pre, post: BlockNorm(
            RMSNormLeaf(pre), RMSNormLeaf(post), residual_scale=0.5, block_scale=2.0, activation="sigmoid")(x, block, g),
            [x, block, g, pre, post])
