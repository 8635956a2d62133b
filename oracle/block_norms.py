"""The norms around a block, in float64 numpy (`omnia_gated_rms_norm` and `omnia_block_norm`,
include/omnia_hip.h)."""

from __future__ import annotations

import numpy as np


def _sigmoid(z):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-z))


def _inverse(x, eps: float):
    return 1.0 / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps)


def gated_rms_norm(x, gate, weight, group: int, eps: float, silu: bool, gate_first: bool):
    """x, gate [rows, width], weight [group] or [width] -> [rows, width]."""
    x, z, weight = (np.asarray(a, dtype=np.float64).reshape(*np.shape(a)[:-1], np.shape(a)[-1] // group, group) for a in (x, gate, weight))
    act = _sigmoid(z) * (z if silu else 1.0)
    y = x * act if gate_first else x
    y = y * _inverse(y, eps) * weight
    return (y if gate_first else y * act).reshape(*y.shape[:-2], y.shape[-2] * group)


def block_norm(x, block, pre, pre_eps: float, post=None, post_eps: float = 0.0, gate=None, sigmoid: bool = False,
               residual_scale: float = 1.0, block_scale: float = 1.0):
    """x, block [rows, hidden] -> (s, its norm, and the absolute terms of s: the scale of its rounding)."""
    x, y = np.asarray(x, dtype=np.float64), np.asarray(block, dtype=np.float64)
    if post is not None:
        y = y * _inverse(y, post_eps) * np.asarray(post, dtype=np.float64)
    if gate is not None:
        gate = np.asarray(gate, dtype=np.float64)
        y = y * (_sigmoid(gate) if sigmoid else gate)
    s = residual_scale * x + block_scale * y
    return s, s * _inverse(s, pre_eps) * np.asarray(pre, dtype=np.float64), (
        np.abs(residual_scale * x) + np.abs(block_scale * y))
