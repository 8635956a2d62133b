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
