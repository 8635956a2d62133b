"""Calls whose grid would come to 2^32 lanes or more, which no launch carries, are refused by their
arguments alone: before a device is asked for, and whatever the pointers are."""

from __future__ import annotations

import ctypes

import pytest

from mlx_omnia_amd.runtime.loader import LinearAttentionCall, call

SOME = 4096   # a pointer, which nothing reads


@pytest.mark.parametrize("rows,width,group", [(1 << 30, 8, 8), (1 << 28, 32, 8), (1 << 29, 72, 72), (1 << 28, 136, 136),
                                              (1 << 27, 264, 264), (1 << 26, 520, 520), (1 << 26, 8192, 8192)])
def test_gated_rms_norm(rows, width, group):
    with pytest.raises(ValueError, match="too many groups for one launch"):
        call("omnia_gated_rms_norm", SOME, width, SOME, width, SOME, group, rows, width, group, 1e-6, 1, 0, SOME, None)


@pytest.mark.parametrize("rows,hidden", [(1 << 26, 8), (1 << 26, 512), (1 << 25, 520), (1 << 24, 1032), (1 << 23, 2056),
                                         (1 << 23, 16384)])
def test_block_norm(rows, hidden):
    with pytest.raises(ValueError, match="too many rows for one launch"):
        call("omnia_block_norm", SOME, SOME, None, 0, 0, None, 0.0, SOME, 1e-6, 1.0, 1.0, rows, hidden, SOME, SOME, None)


@pytest.mark.parametrize("heads,key_dim,value_dim,count", [
    (64, 128, 128, dict(step_count=1 << 16)), (64, 128, 64, dict(step_count=1 << 16)), (4096, 64, 64, dict(step_count=1 << 12)),
    (4096, 128, 128, dict(run_count=1 << 12)), (4096, 64, 64, dict(run_count=1 << 13))])
def test_linear_attention(heads, key_dim, value_dim, count):
    args = LinearAttentionCall(
        queries=SOME, keys=SOME, values=SOME, log_decay=SOME, states=SOME, steps=SOME, runs=SOME, out=SOME,
        query_stride=heads * key_dim, key_stride=heads * key_dim, value_stride=heads * value_dim, decay_stride=0,
        slots=1 << 16, tokens=(1 << 24) - 1, heads=heads, key_heads=heads, key_dim=key_dim, value_dim=value_dim, scale=1.0, **count)
    with pytest.raises(ValueError, match="too many steps or runs for one launch"):
        call("omnia_linear_attention", ctypes.addressof(args), None)
