"""A step of many sequences over one cache of pages: raw q/k/v projections in, context out.

The batch's counterpart of `AttentionStep` (core/kernels/attention/kernel.py: one sequence's,
the reference has no other): the declaration is the same, with a `PagedKVCache` and the layer
of it, and a call names the `PagedBatch` that steps.

- `HipBatchAttentionStep` (`omnia_attention_batch_project`, `omnia_attention_batch`,
  csrc/attention_batch.hip): bf16, head_dim 64 or 128, any number of query heads per kv head,
  with or without gains, a rotary table and sinks, any number of new tokens a sequence. The
  rows that the batch's sequences share are read once for all of them.
- `DefaultBatchAttentionStep` is the Core chain, a sequence at a time in torch ops (fp32). It
  accepts everything, calls that autograd follows among it: gradients of the step's own q, k and v.

The norm, the rotation and mscale are rounded once, as one operation (`AttentionStep` rounds
after each, as its reference does).
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Protocol, runtime_checkable

import torch

from ...runtime import ops
from .._device import hip_device
from ..qkv_rope.atlas import AngleAtlas
from ..qkv_rope.kernel import AngleTable
from ..resolve import record_fallback, resolve
from .pages import PagedBatch, PagedKVCache, _capturing
from .prefill import unfollowed

HEAD_DIMS = (64, 128)


@runtime_checkable
class BatchAttentionStepStrategy(Protocol):
    """A batch's N packed tokens: raw_queries [(1,) N, heads * D], raw_keys and raw_values
    [(1,) N, kv_heads * D] -> the context [N, heads, D], the tokens' rows written."""

    def project(self, batch: PagedBatch, raw_queries: torch.Tensor, raw_keys: torch.Tensor,
                raw_values: torch.Tensor) -> torch.Tensor: ...

    def __call__(self, batch: PagedBatch, raw_queries: torch.Tensor, raw_keys: torch.Tensor,
                 raw_values: torch.Tensor) -> torch.Tensor: ...


def batch_step_applies(heads: int, kv_heads: int, head_dim: int, rotary_pairs: int) -> bool:
    """head_dim 64 or 128, whole groups of query heads, the rotated half in whole lanes."""
    return (head_dim in HEAD_DIMS and kv_heads > 0 and heads > 0 and heads % kv_heads == 0 and heads <= 4096
            and rotary_pairs >= 0 and rotary_pairs % 8 == 0 and 2 * rotary_pairs <= head_dim)


def _check_rows(batch: PagedBatch, raw: torch.Tensor, width: int, name: str) -> None:
    if raw.shape[-2:] != (batch.total, width) or raw.numel() != batch.total * width:
        raise ValueError(f"{name}: expected the batch's {batch.total} tokens of {width}, not {tuple(raw.shape)}")


@dataclass(frozen=True)
class DefaultBatchAttentionStep(BatchAttentionStepStrategy):
    cache: PagedKVCache
    layer: int
    heads: int
    kv_heads: int
    head_dim: int
    scale: float
    query_weight: torch.Tensor | None
    key_weight: torch.Tensor | None
    eps: float
    rotary_pairs: int
    mscale: float
    angles: AngleTable | AngleAtlas | None
    sinks: torch.Tensor | None

    @classmethod
    def build(cls, cache, *, layer, heads, kv_heads, head_dim, scale, dtype, query_weight, key_weight, eps,
              rotary_pairs, mscale, angles, sinks) -> "DefaultBatchAttentionStep":
        return cls(cache, layer, heads, kv_heads, head_dim, scale, query_weight, key_weight, eps, rotary_pairs,
                   mscale, angles, sinks)

    def _positions(self, batch: PagedBatch, device) -> torch.Tensor:
        """Each token's position, from the host's lengths."""
        first = self.cache._rows[batch.index].tolist()
        return torch.cat([torch.arange(n, n + t, device=device) for n, t in zip(first, batch.tokens)])

    def _turn(self, x: torch.Tensor, gain: torch.Tensor | None, rows: torch.Tensor | None) -> torch.Tensor:
        """[N, heads, D] normed and rotated, fp32."""
        x, p = x.float(), self.rotary_pairs
        if gain is not None:
            x = x * torch.rsqrt(x.pow(2).mean(dim=-1, keepdim=True) + self.eps) * gain.float()
        if rows is None:
            return x
        cos, sin = rows[:, None, :p], rows[:, None, p:]
        a, b = x[..., :p] * self.mscale, x[..., p : 2 * p] * self.mscale
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * p :]], dim=-1)

    def _project(self, batch, raw_queries, raw_keys, raw_values):
        """The tokens' queries, and their key and value rows as they were written."""
        d, cache, size = self.head_dim, self.cache, self.cache.page_rows
        _check_rows(batch, raw_queries, self.heads * d, "raw_queries")
        _check_rows(batch, raw_keys, self.kv_heads * d, "raw_keys")
        _check_rows(batch, raw_values, self.kv_heads * d, "raw_values")
        if _capturing(raw_queries.device):
            raise ValueError("batch attention step: only the HIP binding can be captured")
        last = cache.ready(batch)
        at = self._positions(batch, raw_queries.device)
        rows = None
        if self.rotary_pairs:
            table = self.angles(0, last).to(device=raw_queries.device, dtype=torch.float32)
            if table.shape[0] < last:
                raise ValueError(f"position {last - 1} is past the angle table's {table.shape[0]} rows")
            rows = table[at]
        q, k = (self._turn(raw.reshape(batch.total, -1, d), gain, rows)
                for raw, gain in ((raw_queries, self.query_weight), (raw_keys, self.key_weight)))
        whose = torch.repeat_interleave(batch.chosen.long(), batch.rows.long())
        page = cache.tables[whose, at // size].long()
        kind = cache.keys.dtype
        k, v = k.to(kind), raw_values.reshape(batch.total, -1, d).to(kind)
        # The pool itself follows no gradient: rows of earlier steps are constants.
        cache.keys[self.layer, page, :, at % size] = k.detach()
        cache.values[self.layer, page, :, at % size] = v.detach()
        return q.to(raw_queries.dtype), k, v

    def project(self, batch, raw_queries, raw_keys, raw_values):
        return self._project(batch, raw_queries, raw_keys, raw_values)[0]

    def _attend(self, batch: PagedBatch, queries: torch.Tensor, new_keys: torch.Tensor,
                new_values: torch.Tensor) -> torch.Tensor:
        cache, d, kv = self.cache, self.head_dim, self.kv_heads
        group, out, end = self.heads // kv, [], 0
        for s, count in zip(batch.sequences, batch.tokens):
            before, first = int(cache._rows[s]), end
            rows, end = before + count, first + count
            pages = cache.tables[s, : -(-rows // cache.page_rows)].long()
            keys, values = (torch.cat([pool[self.layer, pages].transpose(0, 1).reshape(kv, -1, d)[:, :before],
                                       new[first:end].transpose(0, 1)], dim=1).float()
                            for pool, new in ((cache.keys, new_keys), (cache.values, new_values)))
            q = queries[first:end].float().unflatten(1, (kv, group)).permute(1, 2, 0, 3).reshape(kv, group * count, d)
            scores = (q @ keys.transpose(1, 2).contiguous()).unflatten(1, (group, count)) * self.scale
            seen = (torch.arange(rows, device=q.device)[None]
                    <= torch.arange(before, rows, device=q.device)[:, None])
            scores = scores.masked_fill(~seen, -math.inf)
            if self.sinks is not None:
                sink = self.sinks.float().reshape(kv, group, 1, 1).expand(kv, group, count, 1)
                weights = torch.softmax(torch.cat([sink, scores], dim=-1), dim=-1)[..., 1:]
            else:
                weights = torch.softmax(scores, dim=-1)
            context = (weights.flatten(1, 2) @ values).unflatten(1, (group, count))
            if count > 1 and not bool(torch.isfinite(values).all()):
                # Zero times an infinity that a token does not see is a NaN: such values a token at a time.
                for t in range(count - 1):
                    context[:, :, t] = weights[:, :, t, : before + t + 1] @ values[:, : before + t + 1]
            out.append(context.permute(2, 0, 1, 3).reshape(count, self.heads, d))
        return torch.cat(out).to(queries.dtype)

    def __call__(self, batch, raw_queries, raw_keys, raw_values):
        return self._attend(batch, *self._project(batch, raw_queries, raw_keys, raw_values))


@dataclass(frozen=True, eq=False)
class HipBatchAttentionStep(BatchAttentionStepStrategy):
    core: DefaultBatchAttentionStep
    held: tuple[torch.Tensor, ...]   # the parameters and tables that autograd may follow

    @classmethod
    def build(cls, cache, *, layer, heads, kv_heads, head_dim, scale, dtype, query_weight, key_weight, eps,
              rotary_pairs, mscale, angles, sinks) -> "HipBatchAttentionStep | None":
        if dtype != torch.bfloat16 or cache.keys.dtype != dtype:
            return None
        # The kernels take scale * log2(e), in 32 bits.
        if not 2.0 ** -126 <= scale < 2.0 ** 127:
            return None
        if not batch_step_applies(heads, kv_heads, head_dim, rotary_pairs):
            return None
        weights = [w for w in (query_weight, key_weight) if w is not None]
        if any(w.dtype != dtype or w.numel() != head_dim or not w.is_contiguous() or w.data_ptr() % 16
               for w in weights):
            return None
        if sinks is not None and (sinks.dtype != dtype or sinks.numel() != heads):
            return None
        held = [cache.keys, *weights] + ([sinks] if sinks is not None else [])
        if rotary_pairs:
            if not isinstance(angles, (AngleTable, AngleAtlas)) or angles.pairs != rotary_pairs:
                return None
            table = angles.table() if isinstance(angles, AngleAtlas) else angles
            for rows in (table.cos, table.sin):
                if (rows.dtype != torch.float32 or rows.stride(-1) != 1 or rows.data_ptr() % 16
                        or rows.shape != table.cos.shape or rows.stride() != table.cos.stride() or rows.stride(0) % 4):
                    return None
            held += [table.cos, table.sin]
        if not hip_device(*held):
            return None
        return cls(DefaultBatchAttentionStep.build(
            cache, layer=layer, heads=heads, kv_heads=kv_heads, head_dim=head_dim, scale=scale, dtype=dtype,
            query_weight=query_weight, key_weight=key_weight, eps=eps, rotary_pairs=rotary_pairs, mscale=mscale,
            angles=angles, sinks=sinks),
            (*weights, *(() if sinks is None else (sinks,)),
             *((angles.cos, angles.sin) if rotary_pairs and isinstance(angles, AngleTable) else ())))

    def prepare_capture(self, batch: PagedBatch, steps: int) -> None:
        """Before capturing a step of the batch: the pages of its next `steps` steps, the
        angles they reach and what the kernels read of the batch."""
        rows = self.core.cache.prepare_capture(batch, steps)
        if isinstance(self.core.angles, AngleAtlas) and self.core.rotary_pairs:
            self.core.angles.ensure(rows - 1)
        batch.tiles(self.core.heads // self.core.kv_heads)

    def _plan(self, batch: PagedBatch) -> tuple[ops.BatchStepPlan, int]:
        """The batch's plan of this layer, and the most rows a sequence has in the step."""
        core, cache = self.core, self.core.cache
        last = cache.ready(batch)
        plan, laid = batch.plans.get(self, (None, None))
        # A tensor keeps its identity where a module is moved, or a parameter sharded: its address is asked.
        lies = [t.data_ptr() for t in (cache.keys, cache.values, cache.tables, cache.lengths, *self.held)]
        if plan is None or laid != lies or (core.rotary_pairs and last > plan.angle_rows):
            angles = None
            if core.rotary_pairs:
                table = core.angles
                if isinstance(table, AngleAtlas):
                    if not _capturing(cache.keys.device):
                        table.ensure(last - 1)   # grown past its last row
                    table = table.table()
                angles = table.cos, table.sin
                if table.cos.shape[0] < last:
                    raise ValueError(f"a step that may reach position {last - 1} is past the angle table's "
                                     f"{table.cos.shape[0]} rows")
            plan = ops.BatchStepPlan(
                core.query_weight, core.key_weight, angles, cache.keys[core.layer], cache.values[core.layer],
                cache.tables, cache.lengths, batch.token_map, batch.tiles(core.heads // core.kv_heads),
                heads=core.heads, prefix=batch.prefix, prefix_sequence=batch.sequences[0], scale=core.scale,
                eps=core.eps, mscale=core.mscale, sinks=core.sinks, one_token_each=batch.total == len(batch.sequences))
            batch.plans[self] = plan, lies
        if batch.reach and _capturing(cache.keys.device) and all(plan is not held for held in batch.captured):
            batch.captured.append(plan)   # and with it the angles, should the atlas grow
        return plan, last

    def _followed(self, *raw: torch.Tensor) -> bool:
        """A call that autograd, a transform, a mode or a compiler follows, for the torch ops."""
        if unfollowed(*raw, *self.held):
            return False
        record_fallback(self, self.core)
        return True

    def project(self, batch, raw_queries, raw_keys, raw_values):
        if self._followed(raw_queries, raw_keys, raw_values):
            return self.core.project(batch, raw_queries, raw_keys, raw_values)
        return self._plan(batch)[0].project(raw_queries, raw_keys, raw_values)

    def __call__(self, batch, raw_queries, raw_keys, raw_values):
        if self._followed(raw_queries, raw_keys, raw_values):
            return self.core(batch, raw_queries, raw_keys, raw_values)
        plan, last = self._plan(batch)
        # (What replays that go further reach in all is not known.)
        total = batch.own_total(self.core.heads // self.core.kv_heads) if last == batch.last else 0
        return plan(raw_queries, raw_keys, raw_values, last - batch.prefix, total)


_STRATEGIES = (HipBatchAttentionStep, DefaultBatchAttentionStep)


class BatchAttentionStep(BatchAttentionStepStrategy):
    """A layer's step over a cache of pages: picks its binding once, then forwards every call.

    `step(batch, q, k, v)` writes the tokens' rows of this layer and gives their context; the
    sequences are longer only once the cache has been advanced, after every layer's step.
    `step.project` is its first half, the rows written and the queries [N, heads, D]."""

    def __init__(self, cache: PagedKVCache, *, layer: int, heads: int, kv_heads: int, head_dim: int, scale: float,
                 dtype: torch.dtype, query_weight: torch.Tensor | None = None,
                 key_weight: torch.Tensor | None = None, eps: float = 1e-6, rotary_pairs: int = 0,
                 mscale: float = 1.0, angles: AngleTable | AngleAtlas | None = None, base: float = 0.0,
                 sinks: torch.Tensor | None = None, reference: bool = False) -> None:
        layers, _, cached_heads, _, cached_dim = cache.keys.shape
        if not 0 <= layer < layers:
            raise ValueError(f"BatchAttentionStep: layer {layer} of a cache of {layers}")
        if (cached_heads, cached_dim) != (kv_heads, head_dim) or heads % kv_heads or heads < 1:
            raise ValueError(f"BatchAttentionStep: {heads} heads over {kv_heads} of {head_dim}, in a cache of "
                             f"{cached_heads} of {cached_dim}")
        if rotary_pairs and angles is None:
            if base <= 0.0:
                raise ValueError("BatchAttentionStep: rotary pairs need angles or a base")
            angles = AngleAtlas(rotary_pairs, base=base, device=cache.keys.device)
        self.strategy: BatchAttentionStepStrategy = resolve(
            (DefaultBatchAttentionStep,) if reference else _STRATEGIES, cache, layer=layer, heads=heads,
            kv_heads=kv_heads, head_dim=head_dim, scale=scale, dtype=dtype, query_weight=query_weight,
            key_weight=key_weight, eps=eps, rotary_pairs=rotary_pairs, mscale=mscale, angles=angles, sinks=sinks)

    def prepare_capture(self, batch: PagedBatch, steps: int) -> None:
        """Before capturing the batch's step: how many steps its replays will take (the pages
        and the angles for them are reserved here)."""
        prepare = getattr(self.strategy, "prepare_capture", None)
        if prepare is None:
            raise ValueError("batch attention step: only the HIP binding can be captured")
        prepare(batch, steps)

    def project(self, batch, raw_queries, raw_keys, raw_values):
        return self.strategy.project(batch, raw_queries, raw_keys, raw_values)

    def __call__(self, batch, raw_queries, raw_keys, raw_values):
        return self.strategy(batch, raw_queries, raw_keys, raw_values)
