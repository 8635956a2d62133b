"""What a batch of the linear attention holds, and what its first call waits for."""

from __future__ import annotations

import gc
import weakref

import pytest
import torch

from linear_cases import check, inputs
from mlx_omnia_amd.kernels.linear_attention import HipLinearAttention, LinearAttention, LinearBatch

pytestmark = pytest.mark.gpu


def layer(states, key_heads):
    _, heads, key_dim, value_dim = states.shape
    mixer = LinearAttention(states, heads=heads, key_heads=key_heads, key_dim=key_dim, value_dim=value_dim,
                            scale=key_dim ** -0.5, dtype=torch.bfloat16)
    assert isinstance(mixer.strategy, HipLinearAttention)
    return mixer


@pytest.mark.parametrize("tokens", [[1, 3], [200, 1]])
def test_a_batch_keeps_no_layer_alive(tokens):
    made, _, states, slots = inputs(tokens, 4, 2, 64, 64, device="cuda")
    batch, kept = LinearBatch(slots, tokens), layer(states.clone(), 2)
    kept(batch, **made)
    gc.collect()
    before = torch.cuda.memory_allocated()
    mixer = layer(states.clone(), 2)
    mixer(batch, **made)
    gone = weakref.ref(mixer.strategy)
    del mixer
    gc.collect()
    assert gone() is None and torch.cuda.memory_allocated() == before
    own = kept.strategy.core.states
    before = own.clone()
    check(kept(batch, **made), own, made, None, before, slots, tokens, 0.125)
