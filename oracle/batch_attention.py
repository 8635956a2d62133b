"""A batch's attention over a cache of pages, in float64 numpy, one head of one token at a time.

The layout and the rules are those of `omnia_attention_batch_project` and
`omnia_attention_batch` (include/omnia_hip.h): token (s, j) sits at position lengths[s] + j of
sequence s, whose row r is row r % page_rows of page tables[s][r // page_rows], and sees the
rows up to its own that lie on a page of the pool.
"""

from __future__ import annotations

import numpy as np


def turned(raw, gain, cos, sin, eps: float, mscale: float = 1.0):
    """[heads, D] of one token, normed (with a gain) and rotated by its angles [P] (or None)."""
    x = np.asarray(raw, dtype=np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * np.asarray(gain, dtype=np.float64)
    if cos is None:
        return x
    pairs = len(cos)
    c, s = np.asarray(cos, dtype=np.float64), np.asarray(sin, dtype=np.float64)
    a, b = x[:, :pairs] * mscale, x[:, pairs : 2 * pairs] * mscale
    return np.concatenate([a * c - b * s, a * s + b * c, x[:, 2 * pairs :]], axis=1)


def seen_rows(table, rows: int, pages: int, page_rows: int):
    """(page, row) of the first `rows` rows that lie on a page."""
    at = np.arange(max(rows, 0))
    at = at[at // page_rows < len(table)]
    page = np.asarray(table)[at // page_rows]
    there = (page >= 0) & (page < pages)
    return page[there], at[there] % page_rows


def attend(queries, keys, values, tables, lengths, token_map, scale: float, sinks=None):
    """queries [N, heads, D], keys and values [pages, kv_heads, page_rows, D] -> the context and
    the mean of |v| under the same weights, both [N, heads, D] (the scale of their rounding)."""
    queries = np.asarray(queries, dtype=np.float64)
    pages, kv_heads, page_rows, _ = keys.shape
    group = queries.shape[1] // kv_heads
    out, size = np.zeros_like(queries), np.zeros_like(queries)
    for t, (s, j) in enumerate(token_map):
        if not 0 <= s < len(tables):
            continue
        page, row = seen_rows(tables[s], lengths[s] + j + 1, pages, page_rows)
        for kv in range(kv_heads):
            k = np.asarray(keys[page, kv, row], dtype=np.float64)
            v = np.asarray(values[page, kv, row], dtype=np.float64)
            for h in range(kv * group, (kv + 1) * group):
                score = k @ queries[t, h] * scale
                top = max([*score, *([] if sinks is None else [float(sinks[h])])], default=0.0)
                weight = np.exp(score - top)
                total = weight.sum() + (0.0 if sinks is None else np.exp(float(sinks[h]) - top))
                if total > 0:
                    out[t, h], size[t, h] = weight @ v / total, weight @ np.abs(v) / total
    return out, size
