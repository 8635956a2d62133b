"""Cases of the linear attention shared by its tests: inputs, and the distance to the oracle that
arithmetic allows."""

from __future__ import annotations

import numpy as np
import torch

from oracle.linear_attention import linear_attention as oracle

HALF = 2.0 ** -8     # half a bf16 step, relative
STEP = 2.0 ** -24    # half an fp32 step, relative


def inputs(tokens, heads, key_heads, key_dim, value_dim, *, seed=0, strengths=False, decay="token", device="cpu",
           slots=None, fused=False, dtype=torch.bfloat16):
    """The tensors of a call over sequences of `tokens`, and the slots that they take."""
    gen = torch.Generator().manual_seed(seed)
    n = sum(tokens)
    normal = lambda *shape: torch.randn(shape, generator=gen)  # noqa: E731
    sizes = key_heads * key_dim, key_heads * key_dim, heads * value_dim
    rows = normal(n, sum(sizes)).to(dtype).to(device)
    q, k, v = torch.split(rows, sizes, dim=1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    pool = slots if slots is not None else len(tokens) + 2
    made = dict(queries=q.unflatten(1, (key_heads, key_dim)), keys=k.unflatten(1, (key_heads, key_dim)),
                values=v.unflatten(1, (heads, value_dim)),
                log_decay=(-torch.rand(n, heads, generator=gen) ** 4 * 3).to(device) if decay == "token" else None,
                strengths=torch.rand(n, heads, generator=gen).to(device) if strengths else None)
    fixed = (-torch.rand(heads, generator=gen) * 0.2).to(device) if decay == "head" else None
    states = normal(pool, heads, key_dim, value_dim).to(device)
    order = torch.randperm(pool, generator=gen).tolist()[: len(tokens)]
    return made, fixed, states, order


def wide(t):
    return None if t is None else t.detach().double().cpu().numpy()


def check(context, states, made, fixed, before, slots, tokens, scale):
    """Context and states against the oracle. A term of either sum passes at most three roundings a
    token that comes after it (the decay's, its product's and the sum's), its own products' and the
    sum's over a head (under 256 with the exponential's, whose argument is rounded as well); the
    context's operands are held to 16 bits or more (2^-15 of a term for both), and it is rounded
    once to bf16."""
    gates = fixed if made["log_decay"] is None else made["log_decay"]
    want, left, size, sizes = oracle(wide(made["queries"]), wide(made["keys"]), wide(made["values"]), wide(gates),
                                     wide(made["strengths"]), wide(before), slots, tokens, scale)
    rounds = (3 * max(tokens, default=0) + 256) * STEP
    got = wide(context)
    assert got.shape == want.shape
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(got))
    allowed = HALF * np.abs(want) + (rounds + 2.0 ** -14) * size + 2.0 ** -126
    assert (np.abs(got[fine] - want[fine]) <= allowed[fine]).all()
    now = wide(states)
    fine = np.isfinite(left)
    assert np.array_equal(fine, np.isfinite(now))
    allowed = rounds * sizes + 2.0 ** -126
    assert (np.abs(now[fine] - left[fine]) <= allowed[fine]).all()
