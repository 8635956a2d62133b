"""Inputs of the gated norm and the join of two blocks, and the distance to the oracle that
arithmetic allows."""

from __future__ import annotations

import numpy as np
import torch

from oracle import block_norms as oracle

EPS = 1e-6
HALF = 2.0 ** -8
# What an fp32 chain from the inputs to a result is off by at most, relative: the sum of squares
# (added in a tree, or at most 16 and then a tree: under 40 roundings of 2^-24, halved by the
# root), the root, the reciprocal, the exponential (its argument, up to 88, is rounded as well: 88
# steps, of which a value that small shows little) and six products.
CHAIN = 192 * 2.0 ** -24


def _wide(t):
    return None if t is None else t.detach().double().cpu().numpy()


def gated_case(rows, width, weight_width, *, seed=0, device="cpu"):
    gen = torch.Generator().manual_seed(seed + width)
    x, gate = (torch.randn(rows, width, generator=gen).to(torch.bfloat16).to(device) for _ in range(2))
    return x, gate, (1 + 0.1 * torch.randn(weight_width, generator=gen)).to(torch.bfloat16).to(device)


def check_gated(out, x, gate, weight, group, act, gate_first):
    want = oracle.gated_rms_norm(_wide(x), _wide(gate), _wide(weight), group, EPS, act == "silu", gate_first)
    got = _wide(out)
    assert got.shape == want.shape and out.dtype == torch.bfloat16
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    assert (np.abs(got - want)[fine] <= ((HALF + 2 * CHAIN) * np.abs(want) + 2.0 ** -126)[fine]).all()


def block_case(rows, hidden, gate, post, *, seed=0, device="cpu"):
    gen = torch.Generator().manual_seed(seed + hidden)
    normal = lambda *shape: torch.randn(shape, generator=gen).to(torch.bfloat16).to(device)  # noqa: E731
    x, block = 3 * normal(rows, hidden), normal(rows, hidden)
    g = None if gate is None else normal(hidden) if gate == "row" else normal(rows, hidden)
    pre, behind = 1 + 0.125 * normal(hidden), 1 + 0.125 * normal(hidden)
    return x, block, g, pre, behind if post else None


def check_block(got, x, block, gate, pre, post, act, residual_scale, block_scale, *, pre_eps=EPS, post_eps=1e-5):
    s, n, size = oracle.block_norm(_wide(x), _wide(block), _wide(pre), pre_eps, _wide(post), post_eps, _wide(gate),
                                   act == "sigmoid", residual_scale, block_scale)
    for out, want, terms in ((got[0], s, size), (got[1], n, size * np.abs(n) / np.maximum(np.abs(s), 2.0 ** -126))):
        out = _wide(out)
        assert out.shape == want.shape
        assert (np.abs(out - want) <= HALF * np.abs(want) + 2 * CHAIN * (np.abs(want) + terms) + 2.0 ** -126).all()
