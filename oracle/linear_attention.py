"""Linear attention with a decay for each head, in float64 numpy, a token at a time.

    S_t = exp(g_t) S_{t-1} + w_t k_t v_t^T,   o_t = scale * q_t S_t

for the tokens of each sequence in order (`omnia_linear_attention`, include/omnia_hip.h).
"""

from __future__ import annotations

import numpy as np


def linear_attention(queries, keys, values, log_decay, strengths, states, slots, tokens, scale: float):
    """queries, keys [N, key_heads, DK], values [N, heads, DV], log_decay [N, heads] or [heads],
    strengths [N, heads] or None, states [slots, heads, DK, DV] -> the context, the states behind it
    and, for both, what the same sums of absolute values come to (the scale of their rounding)."""
    q, k, v, states = (np.array(x, dtype=np.float64) for x in (queries, keys, values, states))
    n, heads = v.shape[:2]
    group = heads // k.shape[1]
    g = np.broadcast_to(np.asarray(log_decay, dtype=np.float64), (n, heads))
    w = np.ones((n, heads)) if strengths is None else np.asarray(strengths, dtype=np.float64)
    q, k = np.repeat(q, group, axis=1), np.repeat(k, group, axis=1)
    out, size, sizes = np.zeros_like(v), np.zeros_like(v), np.abs(states)
    at = 0
    with np.errstate(invalid="ignore", over="ignore"):
        for slot, count in zip(slots, tokens):
            for t in range(at, at + count):
                keep = np.exp(g[t])[:, None, None]
                new = k[t][:, :, None] * (w[t][:, None] * v[t])[:, None]
                states[slot] = keep * states[slot] + new
                sizes[slot] = keep * sizes[slot] + np.abs(new)
                out[t] = scale * np.einsum("hk,hkv->hv", q[t], states[slot])
                size[t] = scale * np.einsum("hk,hkv->hv", np.abs(q[t]), sizes[slot])
            at += count
    return out, states, size, sizes
