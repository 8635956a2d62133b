"""Linear attention with a decay for each head: a mixer whose state stands in place of a cache.

    S_t = exp(g_t) S_{t-1} + w_t k_t v_t^T,   o_t = scale * q_t S_t

for each sequence's new tokens in order, S [key_dim, value_dim] fp32 of every head in a pool
`states` [slots, heads, key_dim, value_dim]. It serves mixers whose heads forget at rates of their
own: fixed ones (`decay`), or each token's, as state-space layers have them (the single-token
recurrence of core/kernels/ssm): g = -exp(A_log) softplus(a + dt_bias), which `GateSoftplus`
gives, with the strengths w = softplus(a + dt_bias), which are -g exp(-A_log). It has no term that
corrects a value by what the state holds: the gated delta rule, which
models/qwen3_5/layers/deltanet.py makes the same decays for, is another operator. It stands beside
`AttentionStep` as core/kernels/ssm stands beside core/kernels/attention. One call takes prompts
and steps of one token alike, a batch of any lengths:

    states = torch.zeros(slots, heads, key_dim, value_dim, device="cuda")
    mixer = LinearAttention(states, heads=32, key_heads=16, key_dim=128, value_dim=128,
                            scale=128 ** -0.5, dtype=torch.bfloat16)
    batch = LinearBatch([3, 0], [900, 1])          # 900 new tokens of slot 3, one of slot 0
    o = mixer(batch, q, k, v, g)                   # the states of both, moved on

A fresh sequence's state is zeros and a fork's a copy of its parent's (`states[kid] =
states[parent]`): both are the caller's, on the stream of the calls.

- `HipLinearAttention` (`omnia_linear_attention`, csrc/linear_attention.hip): bf16 rows, heads
  of 64 or 128, any number of heads per key head, fp32 gates and states. A layer that is made
  with `dtype=torch.bfloat16` on the device refuses rows and gates of other types.
- `DefaultLinearAttention` is the Core chain in torch ops, and takes everything, calls that
  autograd follows among it: gradients of the call's own inputs (the pool follows none).

A token sees its own sequence's tokens up to itself, and nothing of the values behind them: an
infinity or a NaN there stays with the tokens from its own on.
"""

from __future__ import annotations

import heapq
import math
from collections.abc import Sequence
from dataclasses import dataclass
from typing import Protocol, runtime_checkable
from weakref import WeakKeyDictionary

import numpy as np
import torch

from ...runtime import ops
from .._device import hip_device
from ..attention.prefill import unfollowed
from ..resolve import record_fallback, resolve

__all__ = ["DefaultLinearAttention", "HipLinearAttention", "LinearAttention", "LinearAttentionStrategy",
           "LinearBatch", "applies"]

DIMS = (64, 128)
CHUNK = 64         # tokens that the kernels and the Core chain take together
STEP_TOKENS = 4    # up to which a sequence is walked a token at a time
MIN_PIECE = 2      # chunks of a piece
PART, PIECE, LAUNCHES = 0.45, 0.8, 1.6


class LinearBatch:
    """The sequences of a call: the slots of their states, each once, and how many new tokens each
    has (none among them). Their rows lie together in the call's tensors, in this order. Made on
    the host and kept as long as the same slots step on, or a graph that took a call of it is
    replayed. Its first call, which is made ahead of a capture, sends its lists to the device on the call's
    stream; calls on other streams wait for them there, and a graph's replays are ordered behind that call."""

    def __init__(self, slots: Sequence[int], tokens: Sequence[int], *, device: torch.device | str = "cuda") -> None:
        self.slots, self.tokens = tuple(int(s) for s in slots), tuple(int(n) for n in tokens)
        if len(self.slots) != len(self.tokens):
            raise ValueError(f"LinearBatch: {len(self.slots)} slots with {len(self.tokens)} token counts")
        if len(set(self.slots)) != len(self.slots) or any(s < 0 for s in self.slots):
            raise ValueError("LinearBatch: a slot is named twice, or negative")
        if any(n < 0 for n in self.tokens):
            raise ValueError("LinearBatch: a negative token count")
        self.total = sum(self.tokens)
        if self.total >= 1 << 24:
            raise ValueError(f"LinearBatch: {self.total} tokens, of at most {(1 << 24) - 1}")
        self.device = torch.device(device)
        # What a layer's binding laid out for the batch, which keeps no layer, nor its pool, alive.
        self.plans: WeakKeyDictionary = WeakKeyDictionary()
        self._lists: dict[tuple[int, int], ops.LinearLists] = {}

    def check(self, states: torch.Tensor) -> None:
        if self.slots and max(self.slots) >= states.shape[0]:
            raise ValueError(f"LinearBatch: slot {max(self.slots)} of a pool of {states.shape[0]}")

    def lists(self, heads: int, places: int) -> ops.LinearLists:
        """What a layer of so many heads, of which the card takes `places` at once, does with each
        sequence, on the device: a token at a time, or in one or several pieces
        (`omnia_linear_attention`'s steps, runs and chains)."""
        held = self._lists.get((heads, places))
        if held is None:
            if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise ValueError("a batch's first call cannot be captured: make one before")
            firsts = np.cumsum(self.tokens, dtype=np.int64) - np.asarray(self.tokens, dtype=np.int64)
            steps, handed_on, last, chains, pieces = [], [], [], [], 0
            short = sum(0 < n <= STEP_TOKENS for n in self.tokens)
            # A launch of their own where they are all there is, or fill the card by themselves.
            apart = short * heads >= places or all(n <= STEP_TOKENS for n in self.tokens)
            longest = piece_chunks([-(-n // CHUNK) for n in self.tokens if n > (STEP_TOKENS if apart else 0)],
                                   max(1, places // heads))
            for slot, first, count in zip(self.slots, firsts.tolist(), self.tokens):
                if count <= STEP_TOKENS and (apart or not count):
                    steps += [(slot, first, count)] if count else []
                    continue
                own = -(-count // CHUNK)
                cut = -(-own // longest)
                size = -(-own // cut) * CHUNK
                cut = -(-count // size)
                for i in range(cut):
                    at, rest = first + i * size, count - i * size
                    (last if i == cut - 1 else handed_on).append(
                        (slot, at, min(size, rest), pieces + i if cut > 1 else -1, (i == 0) + 2 * (i == cut - 1)))
                if cut > 2:
                    chains.append((pieces, cut))
                pieces += cut if cut > 1 else 0
            # The longest first: what is left at the end is short.
            for runs in (handed_on, last):
                runs.sort(key=lambda run: -run[2])
            held = self._lists[heads, places] = ops.LinearLists.of(steps, handed_on, last, chains, pieces, self.device)
        return held


def _in_turn(lengths: list[float], places: int) -> float:
    """When the last of these is done, each taken in this order by the place that is free first."""
    if len(lengths) <= places:
        return max(lengths, default=0)
    free = [0] * places
    for n in lengths:
        heapq.heapreplace(free, free[0] + n)
    return max(free)


def piece_chunks(chunks: list[int], places: int) -> int:
    """How many chunks a piece of these sequences has at most, for the least time of all, in chunks:
    what their contexts take with `places` sequences at a time and, where any is cut, the pieces' own
    parts ahead of them (PART of it) and two launches (LAUNCHES); PIECE for each piece's states."""
    if not chunks:
        return 1
    most, share = max(chunks), sum(chunks) / places
    best, least = most, _in_turn(sorted((n + PIECE for n in chunks), reverse=True), places)
    for longer in (1.0, 1.15, 1.35, 1.6, 2.0, 3.0):
        size = max(MIN_PIECE, math.ceil(share * longer))
        if size >= most:
            break
        cuts = [(-(-n // size), n) for n in chunks]
        runs = [(-(-n // cut), cut) for cut, n in cuts]
        all_pieces = sorted((n + PIECE for n, cut in runs for _ in range(cut)), reverse=True)
        parts = sorted((n + PIECE for n, cut in runs for _ in range(cut - 1)), reverse=True)
        time = _in_turn(all_pieces, places) + PART * _in_turn(parts, places) + LAUNCHES
        if time < least:
            best, least = size, time
    return best


@runtime_checkable
class LinearAttentionStrategy(Protocol):
    """A batch's N packed tokens: queries, keys [N, key_heads, key_dim], values [N, heads, value_dim],
    log_decay and strengths [N, heads] fp32 -> the context [N, heads, value_dim]."""

    def __call__(self, batch: LinearBatch, queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                 log_decay: torch.Tensor | None = None, strengths: torch.Tensor | None = None) -> torch.Tensor: ...


def applies(heads: int, key_heads: int, key_dim: int, value_dim: int) -> bool:
    """Heads of 64 or 128, whole groups of them for a key head."""
    return (key_dim in DIMS and value_dim in DIMS and key_heads > 0 and 0 < heads <= 4096 and heads % key_heads == 0)


@dataclass(frozen=True)
class DefaultLinearAttention(LinearAttentionStrategy):
    states: torch.Tensor
    heads: int
    key_heads: int
    scale: float
    decay: torch.Tensor | None

    @classmethod
    def build(cls, states, *, heads, key_heads, key_dim, value_dim, scale, dtype, decay) -> "DefaultLinearAttention":
        return cls(states, heads, key_heads, scale, decay)

    def _check(self, batch: LinearBatch, queries, keys, values, log_decay, strengths) -> None:
        n, (_, heads, key_dim, value_dim) = batch.total, self.states.shape
        of_keys, of_values = (n, self.key_heads, key_dim), (n, heads, value_dim)
        if queries.shape != of_keys or keys.shape != of_keys or values.shape != of_values:
            raise ValueError(f"linear attention: the batch's {n} tokens are queries and keys {of_keys} and values {of_values}, "
                             f"not {tuple(queries.shape)}, {tuple(keys.shape)} and {tuple(values.shape)}")
        for gates, name in ((log_decay, "log_decay"), (strengths, "strengths")):
            if gates is not None and gates.shape != (n, heads):
                raise ValueError(f"linear attention: {name} {(n, heads)}, not {tuple(gates.shape)}")
        batch.check(self.states)

    def _gates(self, batch: LinearBatch, log_decay: torch.Tensor | None) -> torch.Tensor:
        """[N, heads], fp64: its sums lose nothing of a slow decay behind a fast one."""
        gates = self.decay if log_decay is None else log_decay
        if gates is None:
            raise ValueError("linear attention: neither the layer nor the call has a decay")
        return gates.double().expand(batch.total, self.heads)

    def __call__(self, batch, queries, keys, values, log_decay=None, strengths=None):
        self._check(batch, queries, keys, values, log_decay, strengths)
        kind = torch.promote_types(queries.dtype, self.states.dtype)   # 32 bits or more, as the pool holds them
        group = self.heads // self.key_heads
        q, k = (x.to(kind).repeat_interleave(group, dim=1) for x in (queries, keys))
        v, gates = values.to(kind), self._gates(batch, log_decay)
        if strengths is not None:
            v = v * strengths.to(kind)[..., None]
        # Zero times a value that a token does not see is a NaN where it is not finite: then one at a time.
        chunk = CHUNK if bool(torch.isfinite(v).all()) else 1
        out, end = [], 0
        for slot, count in zip(batch.slots, batch.tokens):
            state = self.states[slot].detach().to(kind, copy=True)   # the pool is written below
            for first in range(end, end + count, chunk):
                mine = slice(first, min(first + chunk, end + count))
                # Never -inf, whose differences are NaN: exp(-1e5) is zero as well.
                to = torch.cumsum(gates[mine].clamp(min=-1e5), dim=0).t()   # [heads, n]
                seen = torch.ones(to.shape[1], to.shape[1], dtype=torch.bool, device=to.device).tril()
                apart = torch.where(seen, to[:, :, None] - to[:, None], -math.inf)
                qs, ks, vs = (x[mine].transpose(0, 1) for x in (q, k, v))
                weight = torch.where(seen, qs @ ks.transpose(1, 2).contiguous(), 0) * torch.exp(apart).to(kind)
                mixed = weight @ vs + (qs @ state) * torch.exp(to).to(kind)[..., None]
                out.append(mixed.transpose(0, 1) * self.scale)
                left = torch.exp(to[:, -1:] - to).to(kind)
                state = state * torch.exp(to[:, -1]).to(kind)[:, None, None] + (
                    ks * left[..., None]).transpose(1, 2).contiguous() @ vs
            if count:
                with torch.no_grad():   # the pool itself follows no gradient
                    self.states[slot] = state.to(self.states.dtype)
            end += count
        return torch.cat(out).to(queries.dtype) if out else torch.zeros_like(values)


@dataclass(frozen=True, eq=False)
class HipLinearAttention(LinearAttentionStrategy):
    core: DefaultLinearAttention

    @classmethod
    def build(cls, states, *, heads, key_heads, key_dim, value_dim, scale, dtype, decay) -> "HipLinearAttention | None":
        if dtype != torch.bfloat16 or states.dtype != torch.float32 or not states.is_contiguous():
            return None
        if not applies(heads, key_heads, key_dim, value_dim) or states.data_ptr() % 16:
            return None
        if decay is not None and (decay.dtype != torch.float32 or not decay.is_contiguous()):
            return None
        if not hip_device(states, *(() if decay is None else (decay,))):
            return None
        return cls(DefaultLinearAttention(states, heads, key_heads, scale, decay))

    def __call__(self, batch, queries, keys, values, log_decay=None, strengths=None):
        core = self.core
        gates = log_decay
        if gates is None:
            gates = core.decay
            if gates is None:
                raise ValueError("linear attention: neither the layer nor the call has a decay")
        elif gates.dim() != 2:
            raise ValueError(f"linear attention: log_decay for every token, not {tuple(gates.shape)}")
        states = core.states
        if not (unfollowed(queries, keys, values, gates, states) if strengths is None
                else unfollowed(queries, keys, values, gates, states, strengths)):
            record_fallback(self, core)
            return core(batch, queries, keys, values, log_decay, strengths)
        plan, at = batch.plans.get(self, (None, 0))
        if plan is None or at != states.data_ptr():   # a pool that was given other memory
            batch.check(states)
            places = ops.linear_attention_places(states, core.key_heads)
            plan = ops.LinearAttentionPlan(states, batch.lists(core.heads, places), batch.total, key_heads=core.key_heads,
                                           scale=core.scale)
            batch.plans[self] = plan, states.data_ptr()
        return plan(queries, keys, values, gates, strengths)


_STRATEGIES = (HipLinearAttention, DefaultLinearAttention)


class LinearAttention(LinearAttentionStrategy):
    """A layer's mixer over its pool of states: picks its binding once, then forwards every call.

    `decay` [heads] is a layer's fixed log decay, for calls that give none of their own."""

    def __init__(self, states: torch.Tensor, *, heads: int, key_heads: int, key_dim: int, value_dim: int, scale: float,
                 dtype: torch.dtype, decay: torch.Tensor | None = None, reference: bool = False) -> None:
        if states.dim() != 4 or tuple(states.shape[1:]) != (heads, key_dim, value_dim):
            raise ValueError(f"LinearAttention: states [slots, {heads}, {key_dim}, {value_dim}], not {tuple(states.shape)}")
        if key_heads < 1 or heads < 1 or heads % key_heads:
            raise ValueError(f"LinearAttention: {heads} heads over {key_heads} key heads")
        if not states.is_floating_point() or states.element_size() < 4:
            raise ValueError(f"LinearAttention: states in 32 bits or more, not {states.dtype}")
        if decay is not None and decay.shape != (heads,):
            raise ValueError(f"LinearAttention: a decay for each of {heads} heads, not {tuple(decay.shape)}")
        self.strategy: LinearAttentionStrategy = resolve(
            (DefaultLinearAttention,) if reference else _STRATEGIES, states, heads=heads, key_heads=key_heads,
            key_dim=key_dim, value_dim=value_dim, scale=scale, dtype=dtype, decay=decay)

    def __call__(self, batch: LinearBatch, queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                 log_decay: torch.Tensor | None = None, strengths: torch.Tensor | None = None) -> torch.Tensor:
        return self.strategy(batch, queries, keys, values, log_decay, strengths)
