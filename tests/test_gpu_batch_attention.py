"""The cache of pages and the batch step on the device, against the float64 oracle.

Tolerances, from the roundings the kernels make (half a step of bf16 is 2^-8 of the value):
- a query or key row is rounded once, after fp32 operations whose errors are a few 2^-24 of
  the head's largest element: 2^-8 |want| + 2^-19 max |head|;
- a context is taken from the kernel's own queries (fp32, of which the product takes 16 bits)
  and pages: the weights are rounded once (2^-8 of the mean of |v| under them) and the result
  once (2^-8 |want|). The fp32 sums
  add less than 2^-12 of that mean: a score is a sum of at most 128 exact products of a total
  size below 64 here, in fp32 (128 halves of 2^-23 times 64 is below 2^-11 at worst and some
  2^-15 in effect, halved by the softmax's normalisation), and exp2 and the merges a few 2^-22.
"""

from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from mlx_omnia_amd.kernels.attention import BatchAttentionStep, HipBatchAttentionStep, PagedKVCache
from mlx_omnia_amd.kernels.qkv_rope import AngleAtlas, AngleTable
from mlx_omnia_amd.kernels.resolve import FALLBACKS
from mlx_omnia_amd.runtime import ops
from oracle.batch_attention import attend, turned
from paged_model import PagedModel, random_calls

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8


def wide(t: torch.Tensor) -> np.ndarray:
    return t.detach().float().cpu().numpy()


class Case:
    """A cache of random pages with the rows of some sequences, a batch of them, a layer."""

    def __init__(self, *, heads, kv_heads, head_dim, page_rows=16, pairs=0, norms=False, sinks=False, prefix=0,
                 own=(1,), tokens=1, layers=2, layer=1, seed=0, spare=float("nan"), mscale=1.0, scale=None):
        rng = np.random.default_rng(seed)
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        counts = [tokens] * len(own) if isinstance(tokens, int) else list(tokens)
        most = prefix + max(o + t for o, t in zip(own, counts)) + 2 * page_rows
        pages = prefix // page_rows + sum(-(-(o + t) // page_rows) + 2 for o, t in zip(own, counts)) + 4
        shape = (layers, pages, kv_heads, page_rows, head_dim)
        self.cache = PagedKVCache(torch.full(shape, spare, dtype=torch.bfloat16, device="cuda"),
                                  torch.full(shape, spare, dtype=torch.bfloat16, device="cuda"),
                                  sequences=len(own) + 3, rows=most)
        # Pages in no order: some are taken first and given back.
        holes = [self.cache.open(page_rows) for _ in range(2)]
        parent = self.cache.open(prefix)
        self.cache.free(holes[:1])
        kids = self.cache.fork(parent, len(own) - 1) if prefix % page_rows == 0 and len(own) > 1 else []
        self.chosen = [parent, *kids]
        for s, more in zip(self.chosen, own):
            self.cache.reserve(s, prefix + more)
        lengths = [prefix + more for more in own]
        # Those rows are the sequences': the cache is taken up again with them.
        tables = self.cache.tables.cpu().numpy()
        held = np.zeros(len(tables), dtype=int)
        held[self.chosen] = lengths
        held[holes[1]] = page_rows
        self.cache = PagedKVCache(self.cache.keys, self.cache.values, tables=tables, lengths=held,
                                  opened=[*self.chosen, holes[1]])
        for s, n in zip(self.chosen, lengths):
            at = torch.arange(n, device="cuda")
            page = self.cache.tables[s, at // page_rows].long()
            for pool in (self.cache.keys, self.cache.values):
                new = self.normal(layers, n, kv_heads, head_dim)
                if s != parent:   # the shared rows are the parent's
                    new[:, :prefix] = pool[:, page[:prefix], :, at[:prefix] % page_rows].transpose(0, 1)
                for i in range(layers):
                    pool[i, page, :, at % page_rows] = new[i]
        self.heads, self.kv_heads, self.head_dim, self.layer = heads, kv_heads, head_dim, layer
        self.scale = head_dim ** -0.5 if scale is None else scale
        self.qw, self.kw = [(1 + 0.2 * self.normal(head_dim).float()).bfloat16() if norms else None for _ in range(2)]
        self.sinks = self.normal(heads) if sinks else None
        self.pairs, self.mscale = pairs, mscale
        theta = rng.uniform(0, 6.3, (most, pairs))
        self.cos, self.sin = (torch.from_numpy(f(theta).astype(np.float32)).cuda() for f in (np.cos, np.sin))
        self.batch = self.cache.batch(self.chosen, tokens=counts)
        self.raw = [self.normal(self.batch.total, n * head_dim) for n in (heads, kv_heads, kv_heads)]
        self.step = self.make(self.cache)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.gen, device="cuda").bfloat16()

    def make(self, cache, **more):
        step = BatchAttentionStep(
            cache, layer=self.layer, heads=self.heads, kv_heads=self.kv_heads, head_dim=self.head_dim,
            scale=self.scale, dtype=torch.bfloat16, query_weight=self.qw, key_weight=self.kw, eps=1e-6,
            rotary_pairs=self.pairs, mscale=self.mscale,
            angles=AngleTable(self.cos, self.sin) if self.pairs else None, sinks=self.sinks, **more)
        if not more:
            assert isinstance(step.strategy, HipBatchAttentionStep)
        return step

    def wide_queries(self):
        """The queries that the step's attention takes, before any rounding."""
        angles = (self.cos, self.sin) if self.pairs else None
        return ops.attention_batch_project(
            *self.raw, self.qw, self.kw, angles, self.cache.keys[self.layer], self.cache.values[self.layer],
            self.cache.tables, self.cache.lengths, self.batch.token_map, heads=self.heads, eps=1e-6,
            mscale=self.mscale, wide_queries=True)

    def check_rows(self, queries, lengths):
        """Queries, and the key and value rows of the batch's tokens, against the oracle."""
        raw = [wide(t) for t in self.raw]
        gains = [None if w is None else wide(w) for w in (self.qw, self.kw)]
        cos, sin = wide(self.cos), wide(self.sin)
        tables, size = self.cache.tables.cpu().numpy(), self.cache.page_rows
        keys, values = wide(self.cache.keys[self.layer]), wide(self.cache.values[self.layer])
        for t, (s, j) in enumerate(self.batch.token_map.cpu().numpy()):
            p = int(lengths[s]) + j
            angles = (cos[p], sin[p]) if self.pairs else (None, None)
            page = tables[s, p // size]
            for got, source, gain in ((wide(queries[t]), raw[0][t], gains[0]),
                                      (keys[page, :, p % size], raw[1][t], gains[1])):
                want = turned(source.reshape(-1, self.head_dim), gain, *angles, 1e-6, self.mscale)
                bound = HALF * np.abs(want) + 2.0 ** -19 * np.abs(want).max(axis=1, keepdims=True)
                assert np.all(np.abs(got - want) <= bound), (t, np.abs(got - want).max())
            assert np.array_equal(values[page, :, p % size], raw[2][t].reshape(-1, self.head_dim))

    def check_context(self, context, queries, lengths, rows=None):
        pick = np.arange(self.batch.total) if rows is None else np.asarray(rows)
        sinks = None if self.sinks is None else wide(self.sinks)
        want, size = attend(wide(queries)[pick], wide(self.cache.keys[self.layer]), wide(self.cache.values[self.layer]),
                            self.cache.tables.cpu().numpy(), lengths, self.batch.token_map.cpu().numpy()[pick],
                            self.scale, sinks)
        bad = np.abs(wide(context)[pick] - want) > HALF * np.abs(want) + (HALF + 2.0 ** -12) * size
        assert not bad.any(), (int(bad.sum()), bad.size, np.argwhere(bad)[:4].tolist())

    def check(self, rows=None):
        before = [p[1 - self.layer].clone() for p in (self.cache.keys, self.cache.values)]
        lengths = self.cache.lengths.cpu().numpy()
        queries = self.step.project(self.batch, *self.raw)
        self.check_rows(queries, lengths)
        rounded, queries = queries, self.wide_queries()
        assert torch.equal(rounded, queries.bfloat16())
        context = self.step(self.batch, *self.raw)
        assert context.shape == (self.batch.total, self.heads, self.head_dim)
        self.check_context(context, queries, lengths, rows)
        again = self.step(self.batch, *self.raw)
        assert torch.equal(context.view(torch.int16), again.view(torch.int16))   # the same to the last bit
        for kept, pool in zip(before, (self.cache.keys, self.cache.values)):
            assert torch.equal(kept.view(torch.int16), pool[1 - self.layer].view(torch.int16))
        return context


GEOMETRIES = [
    # one token each: groups of 1 to 16, both head sizes, odd batches, every page size
    dict(heads=2, kv_heads=2, head_dim=128, own=(1,)),
    dict(heads=8, kv_heads=2, head_dim=128, pairs=64, norms=True, own=(0,)),
    dict(heads=8, kv_heads=2, head_dim=128, pairs=64, norms=True, prefix=208, own=(1, 20)),
    dict(heads=32, kv_heads=8, head_dim=128, pairs=64, norms=True, page_rows=64, prefix=640, own=(3, 70, 0, 128, 64)),
    dict(heads=16, kv_heads=2, head_dim=64, pairs=32, sinks=True, prefix=48, own=tuple(range(0, 33, 3))),
    dict(heads=9, kv_heads=3, head_dim=64, pairs=8, norms=True, page_rows=32, prefix=2016, own=(5, 300)),
    dict(heads=5, kv_heads=1, head_dim=128, pairs=32, page_rows=128, prefix=1024, own=(17, 0, 130), mscale=1.3),
    dict(heads=16, kv_heads=1, head_dim=128, page_rows=256, prefix=256, own=(255, 256, 257, 1)),
    dict(heads=64, kv_heads=8, head_dim=64, pairs=32, sinks=True, page_rows=16, prefix=2000, own=(333, 90, 4)),
    dict(heads=4, kv_heads=1, head_dim=128, page_rows=16, prefix=0, own=(5000,)),
    dict(heads=8, kv_heads=8, head_dim=64, page_rows=16, prefix=16, own=tuple((i * 37) % 61 for i in range(70))),
    # prompts: one and several tokens, a prompt into an empty sequence, tiles that end anywhere
    dict(heads=8, kv_heads=2, head_dim=128, pairs=64, norms=True, own=(0,), tokens=2),
    dict(heads=8, kv_heads=2, head_dim=128, pairs=64, norms=True, own=(0,), tokens=200),
    dict(heads=8, kv_heads=2, head_dim=64, sinks=True, page_rows=32, prefix=320, own=(0, 7, 33), tokens=(40, 1, 129)),
    dict(heads=12, kv_heads=4, head_dim=128, pairs=64, page_rows=64, prefix=128, own=(65, 0), tokens=(3, 70)),
    dict(heads=16, kv_heads=1, head_dim=128, page_rows=16, prefix=0, own=(777,), tokens=33),
    dict(heads=129, kv_heads=1, head_dim=64, page_rows=16, prefix=32, own=(3, 9), tokens=(2, 3)),
]


# What a plan chooses by: shared rows read once, for tiles of some rows, of many and of many tokens;
# own rows alone, past the caches, a tile of more than 16 rows among them; steps beside prompts.
PLANS = [
    dict(heads=8, kv_heads=2, head_dim=128, pairs=64, norms=True, prefix=640, own=(5, 0, 17), tokens=(2, 1, 3)),
    dict(heads=16, kv_heads=2, head_dim=64, sinks=True, prefix=1008, own=(3, 30, 9, 1, 70, 64), tokens=(1, 9, 1, 1, 17, 2)),
    dict(heads=32, kv_heads=2, head_dim=128, page_rows=64, prefix=704, own=tuple(range(12)), tokens=2),
    dict(heads=16, kv_heads=4, head_dim=128, page_rows=32, prefix=1024, own=tuple((i * 29) % 130 for i in range(40))),
    dict(heads=8, kv_heads=1, head_dim=64, page_rows=16, prefix=4000, own=(1, 2, 3, 4), tokens=(1, 1, 1, 5)),
    dict(heads=16, kv_heads=8, head_dim=64, pairs=32, sinks=True, page_rows=256, prefix=0, own=(3000,) * 21 + (0, 1, 256)),
    dict(heads=24, kv_heads=8, head_dim=128, page_rows=64, prefix=0, own=(2900, 17, 0) + (2750,) * 21,
         tokens=(1, 20, 6) + (1,) * 21),
    dict(heads=24, kv_heads=8, head_dim=128, pairs=32, norms=True, page_rows=64, prefix=0,
         own=(2900, 0, 255, 256) + (2751,) * 20),
    dict(heads=16, kv_heads=4, head_dim=128, pairs=64, page_rows=64, prefix=0, own=(700, 0, 1500, 9, 64), tokens=(1, 300, 1, 2, 75)),
    dict(heads=16, kv_heads=4, head_dim=64, page_rows=16, prefix=320, own=(700, 0, 9, 64), tokens=(1, 150, 1, 1)),
]


@pytest.mark.parametrize("case", PLANS, ids=lambda c: "-".join(f"{v}" for v in c.values()).replace(" ", ""))
def test_plans(case):
    made = Case(**case)
    made.check(None if made.batch.total * made.heads < 2000 else np.arange(0, made.batch.total, 7))


# Every way that a row's weights go into their product: a wave's own rows with and without the
# prologue's launch, shared rows for many tokens and for few, own rows alone, prompts.
WEIGHTS = [
    dict(heads=8, kv_heads=2, head_dim=128, pairs=64, norms=True, prefix=64, own=(0, 1, 5, 20)),
    dict(heads=16, kv_heads=2, head_dim=64, pairs=8, own=(0, 1, 2, 3, 40)),
    dict(heads=16, kv_heads=4, head_dim=128, prefix=1024, own=tuple((i * 29) % 130 for i in range(40))),
    dict(heads=8, kv_heads=8, head_dim=64, prefix=640, own=tuple(range(0, 61)) + (9,) * 30, sinks=True),
    dict(heads=24, kv_heads=8, head_dim=128, pairs=32, norms=True, page_rows=64, own=(0, 1, 2, 3) + (2751,) * 20),
    dict(heads=24, kv_heads=8, head_dim=64, page_rows=64, own=(0, 1, 2, 3) + (2751,) * 20, tokens=(2, 1, 1, 1) + (1,) * 20),
    dict(heads=8, kv_heads=2, head_dim=128, pairs=64, norms=True, own=(0,), tokens=200),
    dict(heads=8, kv_heads=2, head_dim=64, sinks=True, page_rows=32, own=(0, 7, 33), tokens=(40, 1, 129)),
]


@pytest.mark.parametrize("case", WEIGHTS, ids=lambda c: "-".join(f"{v}" for v in c.values()).replace(" ", "")[:60])
def test_weights_are_held_in_sixteen_bits(case):
    """What remains beside the result's own rounding, in parts of the mean of |v|:
    - a weight is cut to 8 bits, which leaves less than 2^-7 of it, and the rest rounded by at
      most 2^-8 of itself: 2^-15;
    - fp32 queries are rounded to 8 bits, what that leaves (2^-8 at most) to 8 more: 2^-16 of
      each, and a score's 128 products are summed in fp32 (128 halves of 2^-23, 2^-17): with
      |q . k| of the absolutes at most ||q|| ||k||, a score is off by (2^-16 + 2^-17) of that times
      the scale, the weight by as much of itself, and so is the sum that it is divided by;
    - n rows summed in fp32: n 2^-24 in the context and in the sum of the weights;
    - exp2, the merges and the products of fp32 around them, of 2^-22 or less each: 2^-18."""
    made = Case(**case, scale=0.02)
    lengths = made.cache.lengths.cpu().numpy()
    context, queries = made.step(made.batch, *made.raw), made.wide_queries()
    token_map, sinks = made.batch.token_map.cpu().numpy(), None if made.sinks is None else wide(made.sinks)
    keys, values = wide(made.cache.keys[made.layer]), wide(made.cache.values[made.layer])
    tables = made.cache.tables.cpu().numpy()
    seen = lengths[token_map[:, 0]] + token_map[:, 1] + 1
    pick = np.flatnonzero((seen <= 200) | (np.arange(len(seen)) % 5 == 0))
    longest = np.sqrt(np.nanmax((keys.astype(np.float64) ** 2).sum(axis=-1)))
    rounded = queries.bfloat16()
    alone = ops.attention_batch(rounded, made.cache.keys[made.layer], made.cache.values[made.layer], made.cache.tables,
                                made.cache.lengths, made.batch.token_map, made.batch.tiles(made.heads // made.kv_heads),
                                prefix=made.batch.prefix, prefix_sequence=made.chosen[0],
                                own_rows=int(seen.max()) - made.batch.prefix, scale=made.scale, sinks=made.sinks)
    for got, q, query_bits in ((context, queries, 2.0 ** -16), (alone, rounded, 0.0)):
        want, size = attend(wide(q)[pick], keys, values, tables, lengths, token_map[pick], made.scale, sinks)
        score = np.linalg.norm(wide(q)[pick], axis=-1, keepdims=True) * longest * made.scale
        bound = (2.0 ** -15 + 2 * (query_bits + 2.0 ** -17) * score
                 + 2 * seen[pick][:, None, None] * 2.0 ** -24 + 2.0 ** -18)
        bad = np.abs(wide(got)[pick] - want) > HALF * np.abs(want) + bound * size
        assert not bad.any(), (int(bad.sum()), bad.size, np.argwhere(bad)[:4].tolist())


@pytest.mark.parametrize("case", [c for c in PLANS + GEOMETRIES if c.get("tokens", 1) == 1],
                         ids=lambda c: "-".join(f"{v}" for v in c.values()).replace(" ", ""))
def test_a_step_writes_its_rows_and_no_others(case):
    """Without the prologue's own launch ahead of it, which would have written them."""
    made = Case(**case)
    cache, size, d = made.cache, made.cache.page_rows, made.head_dim
    before = [p.clone() for p in (cache.keys, cache.values)]
    lengths = cache.lengths.cpu().numpy()
    context = made.step(made.batch, *made.raw)   # which takes pages where a sequence's are full
    tables = cache.tables.cpu().numpy()
    raw, gain = [wide(t) for t in made.raw], None if made.kw is None else wide(made.kw)
    cos, sin = wide(made.cos), wide(made.sin)
    for t, (s, j) in enumerate(made.batch.token_map.cpu().numpy()):
        p = int(lengths[s]) + j
        angles = (cos[p], sin[p]) if made.pairs else (None, None)
        page, row = int(tables[s, p // size]), p % size
        key, value = (wide(pool[made.layer, page, :, row]) for pool in (cache.keys, cache.values))
        want = turned(raw[1][t].reshape(-1, d), gain, *angles, 1e-6, made.mscale)
        assert np.all(np.abs(key - want) <= HALF * np.abs(want) + 2.0 ** -19 * np.abs(want).max(axis=1, keepdims=True))
        assert np.array_equal(value, raw[2][t].reshape(-1, d))
        for pool, was in zip((cache.keys, cache.values), before):
            was[made.layer, page, :, row] = pool[made.layer, page, :, row]
    for pool, was in zip((cache.keys, cache.values), before):
        assert torch.equal(pool.view(torch.int16), was.view(torch.int16))
    if made.batch.total * made.heads < 2000:
        made.check_context(context, made.wide_queries(), lengths)


def test_values_that_are_not_finite_among_own_rows_alone():
    """Rows behind a token's own are not there for it, whatever they hold, 16 rows of a tile at a time."""
    case = Case(heads=24, kv_heads=8, head_dim=128, page_rows=64, own=(2900, 17) + (2750,) * 21, tokens=(1, 20) + (1,) * 21)
    clean = case.step(case.batch, *case.raw)
    v = case.raw[2].view(case.batch.total, 8, 128)
    v[9, 3, 40] = float("inf")
    out = case.step(case.batch, *case.raw)
    touched = torch.zeros_like(out, dtype=torch.bool)
    touched[9:21, 9:12, 40] = True
    assert torch.equal(out[~touched], clean[~touched]) and (out[touched] == float("inf")).all()


@pytest.mark.parametrize("case", GEOMETRIES, ids=lambda c: "-".join(f"{v}" for v in c.values()).replace(" ", ""))
def test_step(case):
    made = Case(**case)
    made.check(None if made.batch.total * made.heads < 2000 else np.arange(0, made.batch.total, 7))


def test_rows_in_use_may_hold_anything_where_nobody_looks():
    """Pages and page ends nobody holds are NaN in every case here; infinities as well."""
    for spare in (float("inf"), -3.0e38):
        Case(heads=8, kv_heads=2, head_dim=128, prefix=96, own=(5, 1, 40), tokens=(1, 3, 1), spare=spare).check()


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_a_value_that_is_not_finite_reaches_only_who_sees_it(head_dim, value):
    case = Case(heads=8, kv_heads=2, head_dim=head_dim, prefix=32, own=(9, 3), tokens=(50, 20))
    clean = case.step(case.batch, *case.raw)
    v = case.raw[2].view(case.batch.total, 2, head_dim)
    v[30, 1, 5] = value
    v[60, 0, 7] = value
    out = case.step(case.batch, *case.raw)
    touched = torch.zeros_like(out, dtype=torch.bool)
    touched[30:50, 4:, 5] = True
    touched[60:70, :4, 7] = True
    assert torch.equal(out[~touched], clean[~touched])
    assert (torch.isnan if value != value else lambda t: t == value)(out[touched]).all()


def test_infinite_sinks_and_scores():
    case = Case(heads=4, kv_heads=2, head_dim=64, prefix=16, own=(3, 5), sinks=True)
    case.sinks[0], case.sinks[1] = -float("inf"), 80.0
    case.step = case.make(case.cache)
    out = case.check()
    assert out[:, 1].abs().max() < 1e-20   # e^80 in the denominator
    large = Case(heads=4, kv_heads=2, head_dim=64, prefix=16, own=(30, 5), scale=8.0)
    large.check()   # scores of some hundreds: nearly one weight a row


@pytest.mark.parametrize("prefix", [64, 640])
def test_tokens_of_no_sequence_and_pages_of_no_pool(prefix):
    case = Case(heads=8, kv_heads=2, head_dim=128, page_rows=16, prefix=prefix, own=(40, 40, 40))
    cache, batch = case.cache, case.batch
    queries = case.step.project(batch, *case.raw)
    tables, token_map = cache.tables.clone(), batch.token_map.clone()
    s = case.chosen[1]
    first = prefix // 16
    tables[s, first] = -1                 # the first rows of one sequence's own are nowhere
    tables[s, first + 1] = cache.pages    # nor are the next
    tables[case.chosen[2], first + 2] = -7
    tables[case.chosen, 1] = -1           # nor 16 of the shared ones
    token_map[0, 0] = cache.tables.shape[0] + 5
    # The second token's sequence gives the shared rows.
    token_map[[0, 1]] = token_map[[1, 0]]
    tiles = batch.tiles(4).clone()
    tiles[:, 2] = token_map[:, 0]
    lengths = cache.lengths.cpu().numpy()
    out = ops.attention_batch(queries, cache.keys[1], cache.values[1], tables, cache.lengths, token_map, tiles,
                              prefix=prefix, prefix_sequence=s, own_rows=41, scale=case.scale)
    assert (out[1] == 0).all()
    want, size = attend(wide(queries), wide(cache.keys[1]), wide(cache.values[1]), tables.cpu().numpy(), lengths,
                        token_map.cpu().numpy(), case.scale)
    assert np.all(np.abs(wide(out) - want) <= HALF * np.abs(want) + (HALF + 2.0 ** -12) * size)
    # Nothing is written for them either.
    before = cache.keys.clone()
    gone = torch.full_like(cache.tables, -1)
    ops.attention_batch_project(*case.raw, None, None, None, cache.keys[1], cache.values[1], gone, cache.lengths,
                                batch.token_map, heads=8, eps=1e-6)
    assert torch.equal(before.view(torch.int16), cache.keys.view(torch.int16))


@pytest.mark.parametrize("prefix,one_each", [(64, True), (640, True), (640, False)])
def test_a_step_with_rows_that_are_nowhere(prefix, one_each):
    """A new row without a page is not stored and not seen; one of no sequence is zeros, and no page changes."""
    case = Case(heads=8, kv_heads=2, head_dim=128, pairs=64, norms=True, page_rows=16, prefix=prefix, own=(40, 32, 40, 3))
    cache, batch, layer = case.cache, case.batch, case.layer
    cache.ready(batch)
    tables, token_map, tiles = cache.tables.clone(), batch.token_map.clone(), batch.tiles(4).clone()
    lengths = cache.lengths.cpu().numpy()
    tables[case.chosen[1], (prefix + 32) // 16] = -1              # where its new row would be
    tables[case.chosen[0], prefix // 16 + 1] = cache.pages + 3    # some of its own rows
    token_map[2, 0], tiles[2, 2] = -1, -1
    good = case.wide_queries()   # which writes every row where it belongs
    before = [p.clone() for p in (cache.keys, cache.values)]
    plan = ops.BatchStepPlan(case.qw, case.kw, (case.cos, case.sin), cache.keys[layer], cache.values[layer], tables,
                             cache.lengths, token_map, tiles, heads=8, prefix=prefix, prefix_sequence=case.chosen[3],
                             scale=case.scale, eps=1e-6, one_token_each=one_each)
    raw = [t + 1 for t in case.raw]   # other rows than those in the pages by now
    out = plan(*raw, 41)
    assert (out[2] == 0).all()
    for pool, was in zip((cache.keys, cache.values), before):
        for t in (0, 3):
            s = case.chosen[t]
            p = int(lengths[s])
            page = int(tables[s, p // 16])
            assert not torch.equal(pool[layer, page, :, p % 16], was[layer, page, :, p % 16])
            was[layer, page, :, p % 16] = pool[layer, page, :, p % 16]
        assert torch.equal(pool.view(torch.int16), was.view(torch.int16))
    spare = [p.clone() for p in (cache.keys[layer], cache.values[layer])]
    queries = ops.attention_batch_project(*raw, case.qw, case.kw, (case.cos, case.sin), *spare, cache.tables, cache.lengths,
                                          batch.token_map, heads=8, eps=1e-6, wide_queries=True)
    assert queries.shape == good.shape
    want, size = attend(wide(queries), wide(cache.keys[layer]), wide(cache.values[layer]), tables.cpu().numpy(), lengths,
                        token_map.cpu().numpy(), case.scale)
    assert np.all(np.abs(wide(out) - want) <= HALF * np.abs(want) + (HALF + 2.0 ** -12) * size)


@pytest.mark.parametrize("prefix,own", [(160, (9, 4, 1)), (640, (9, 4, 1)), (1600, (9, 4, 1, 30) * 4)])
def test_sequences_shorter_than_the_shared_rows(prefix, own):
    """A plan that is not the cache's own: a sequence that ends inside the shared rows sees its
    rows of them and no more."""
    case = Case(heads=8, kv_heads=2, head_dim=128, page_rows=16, prefix=prefix, own=own)
    cache, batch = case.cache, case.batch
    queries = case.step.project(batch, *case.raw)
    lengths = cache.lengths.clone()
    lengths[case.chosen[1]], lengths[case.chosen[2]] = prefix // 2 - 10, -1
    out = ops.attention_batch(queries, cache.keys[1], cache.values[1], cache.tables, lengths, batch.token_map,
                              batch.tiles(4), prefix=prefix, prefix_sequence=case.chosen[0], own_rows=31,
                              scale=case.scale)
    want, size = attend(wide(queries), wide(cache.keys[1]), wide(cache.values[1]), cache.tables.cpu().numpy(),
                        lengths.cpu().numpy(), batch.token_map.cpu().numpy(), case.scale)
    assert (out[2] == 0).all()
    assert np.all(np.abs(wide(out) - want) <= HALF * np.abs(want) + (HALF + 2.0 ** -12) * size)


@pytest.mark.parametrize("case", [
    dict(heads=4, kv_heads=1, head_dim=128, pairs=64, page_rows=256, own=(0,), tokens=9001),
    dict(heads=16, kv_heads=4, head_dim=64, norms=True, page_rows=64, prefix=5120, own=(900, 0), tokens=(1, 4000)),
    dict(heads=8, kv_heads=1, head_dim=64, sinks=True, page_rows=128, own=(70001,))], ids=["prompt", "beside", "long"])
def test_long_ones(case):
    made = Case(**case, layers=2)
    made.check(np.unique(np.linspace(0, made.batch.total - 1, 9).astype(int)))


@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 128), (24, 2, 128), (40, 2, 64), (70, 5, 128), (70, 7, 64),
                                                     (60, 2, 128), (120, 4, 64)])
def test_prompts_of_many_tokens_into_the_pages(heads, kv_heads, head_dim):
    """One to four heads in turn, and heads that do not fill the last of them."""
    case = Case(heads=heads, kv_heads=kv_heads, head_dim=head_dim, pairs=head_dim // 4, norms=True, page_rows=32,
                prefix=32, own=(3, 40), tokens=(600, 501), layers=2, layer=0)
    case.check_rows(case.step.project(case.batch, *case.raw), case.cache.lengths.cpu().numpy())


def test_raw_rows_are_read_where_they_lie():
    case = Case(heads=8, kv_heads=2, head_dim=128, pairs=64, norms=True, prefix=32, own=(5, 9, 2), tokens=(1, 4, 2))
    want = case.step(case.batch, *case.raw)
    fused = torch.cat(case.raw, dim=1)
    parts = torch.split(fused, [1024, 256, 256], dim=1)
    assert torch.equal(case.step(case.batch, *parts), want)
    assert torch.equal(case.step(case.batch, *(p[None] for p in parts)), want)
    odd = [torch.cat([p.new_zeros(p.shape[0], 3), p], dim=1)[:, 3:] for p in parts]
    assert torch.equal(case.step(case.batch, *odd), want)


def test_reference_and_kernels_agree():
    case = Case(heads=8, kv_heads=2, head_dim=64, pairs=32, norms=True, sinks=True, prefix=64, own=(33, 2), tokens=(5, 9))
    want = case.make(case.cache, reference=True)(case.batch, *case.raw)
    got = case.step(case.batch, *case.raw)
    # The queries may round to either side of a half step, once more than the kernel alone.
    assert (got.float() - want.float()).abs().max() <= 4 * HALF * want.float().abs().max()


def test_a_call_that_autograd_follows_runs_in_torch():
    case = Case(heads=8, kv_heads=2, head_dim=64, prefix=16, own=(3, 4))
    q = case.raw[0].clone().requires_grad_()
    before = dict(FALLBACKS)
    case.step(case.batch, q, *case.raw[1:]).float().sum().backward()
    assert q.grad is not None and torch.isfinite(q.grad).all()
    assert FALLBACKS != before


def test_steps_that_are_captured():
    """A step and its advance, captured once and replayed, with eager work between the replays,
    against the same steps taken eagerly; a page boundary on the way, and another graph."""
    case = Case(heads=8, kv_heads=2, head_dim=128, pairs=64, norms=True, prefix=64, own=(10, 25, 14))
    twin = PagedKVCache(case.cache.keys.clone(), case.cache.values.clone(), tables=case.cache.tables.cpu().numpy(),
                        lengths=case.cache.lengths.cpu().numpy(), opened=[*case.chosen, 1])
    steps = 9
    inputs = [[torch.empty_like(t).normal_(generator=case.gen) for t in case.raw] for _ in range(steps)]
    eager, eager_batch = case.make(twin), twin.batch(case.chosen)
    want = []
    for raw in inputs:
        want.append(eager(eager_batch, *raw))
        twin.advance(eager_batch)
    step, batch, cache = case.step, case.batch, case.cache
    with pytest.raises(ValueError):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(batch, *case.raw)
    torch.cuda.synchronize()
    step.prepare_capture(batch, steps)
    graphs = []
    for advancing in (True, False):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(batch, *case.raw)
            if advancing:
                cache.advance(batch)
        graphs.append((graph, out))
    torch.cuda.synchronize()
    assert cache.rows(case.chosen[0]) == 74
    for raw, expected in zip(inputs, want):
        for held, new in zip(case.raw, raw):
            held.copy_(new)
        graphs[1][0].replay()   # the same step without the advance, from the other graph
        torch.empty(1000, device="cuda").normal_().sum().item()
        graphs[0][0].replay()
        assert torch.equal(graphs[1][1], graphs[0][1])
        # The captured plan cuts the keys for all the rows it was prepared for.
        assert (graphs[0][1].float() - expected.float()).abs().max() <= 4 * HALF * expected.float().abs().max()
    cache.account(batch, steps)
    assert torch.equal(cache.lengths, twin.lengths)
    for s in case.chosen:
        n = cache.rows(s)
        at = torch.arange(n, device="cuda")
        # Pages reserved ahead are others than those taken a step at a time.
        mine, theirs = (c.keys[1, c.tables[s, at // 16].long(), :, at % 16] for c in (cache, twin))
        assert torch.equal(mine, theirs)
    for raw in inputs[:1]:
        assert torch.equal(step(batch, *raw), eager(eager_batch, *raw))


def test_a_fork_between_replays_and_their_account():
    """Its children have the rows that the host has counted, on the device as well, and step on
    as those of a fork ahead of the replays."""
    case = Case(heads=8, kv_heads=2, head_dim=64, pairs=32, prefix=0, own=(21,))
    cache, batch, step = case.cache, case.batch, case.step
    cache.free(1)   # the case's own, for its slot
    step.prepare_capture(batch, 3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(batch, *case.raw)
        cache.advance(batch)
    (early,) = cache.fork(case.chosen[0])
    for _ in range(3):
        graph.replay()
        torch.empty(1000, device="cuda").normal_().sum().item()
    late = [*cache.fork(case.chosen[0]), *cache.fork(case.chosen[0], share=False)]
    assert cache.lengths[[early, *late, case.chosen[0]]].tolist() == [21, 21, 21, 24]
    assert [cache.rows(s) for s in (early, *late)] == [21] * 3
    cache.account(batch, 3)
    assert cache.rows(case.chosen[0]) == 24 and cache.lengths[[early, *late]].tolist() == [21] * 3
    raw = [t + 1 for t in case.raw]
    want = step(cache.batch([early]), *raw)
    for kid in late:
        assert torch.equal(step(cache.batch([kid]), *raw), want)


def test_a_step_is_not_captured_for_fewer_rows_than_it_will_have():
    case = Case(heads=8, kv_heads=2, head_dim=64, prefix=16, own=(3, 4))
    cache, batch, step = case.cache, case.batch, case.step
    step.prepare_capture(batch, 1)
    step(batch, *case.raw)
    cache.advance(batch)   # the one step that was prepared for
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device="cuda")
        with pytest.raises(ValueError, match="prepare_capture"):
            step(batch, *case.raw)
    torch.cuda.synchronize()


def test_a_graph_keeps_the_angles_it_was_captured_with():
    """The atlas grows, for another step, while a graph that reads its first rows lives."""
    case = Case(heads=8, kv_heads=2, head_dim=64, prefix=16, own=(3, 4))
    atlas = AngleAtlas(32, base=1e4, rows=64, device="cuda")
    step = BatchAttentionStep(case.cache, layer=1, heads=8, kv_heads=2, head_dim=64, scale=0.1, dtype=torch.bfloat16,
                              rotary_pairs=32, angles=atlas)
    want = step(case.batch, *case.raw)
    step.prepare_capture(case.batch, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(case.batch, *case.raw)
    assert len(case.batch.captured) == 1
    atlas.ensure(5000)
    case.batch.plans.clear()
    for _ in range(3):
        filler = [torch.full((64, 64), 3.0, device="cuda") for _ in range(50)]   # where freed rows would lie
        graph.replay()
        assert torch.equal(out, want) and len(filler) == 50
        assert torch.equal(step(case.batch, *case.raw), want)


def test_tensors_that_were_given_other_memory():
    """Gains, sinks, angles and the pool of a batch that steps on, moved as a module moves its
    parameters, with other numbers where they were; and sinks that do not lie together."""
    case = Case(heads=8, kv_heads=2, head_dim=64, pairs=32, norms=True, sinks=True, prefix=64, own=(3, 40, 9))
    apart = torch.stack([case.sinks, case.sinks + 1], dim=1)
    loose = BatchAttentionStep(case.cache, layer=case.layer, heads=8, kv_heads=2, head_dim=64, scale=case.scale,
                               dtype=torch.bfloat16, query_weight=case.qw, key_weight=case.kw, rotary_pairs=32,
                               angles=AngleTable(case.cos, case.sin), sinks=apart[:, 0])
    assert isinstance(loose.strategy, HipBatchAttentionStep)
    want, other = case.step(case.batch, *case.raw), loose(case.batch, *case.raw)
    assert torch.equal(other, want)
    held = []
    for t in (case.qw, case.kw, case.sinks, case.cos, case.sin, case.cache.keys, case.cache.values, case.cache.tables,
              case.cache.lengths):
        held.append(t.data)
        t.data = t.data.clone()
        if t.is_floating_point():
            held[-1].fill_(7.0)
        assert torch.equal(case.step(case.batch, *case.raw), want)
    table = case.cache.tables.clone()
    kids = case.cache.fork(case.chosen[1], 2)
    assert torch.equal(case.cache.tables[kids[0], :4], table[case.chosen[1], :4])
    assert (held[-2] == table).all()   # the ones that were left
    assert torch.equal(case.step(case.batch, *case.raw), want)
    apart[:, 0] += 2
    case.sinks += 2
    assert torch.equal(loose(case.batch, *case.raw), case.step(case.batch, *case.raw))
    assert not torch.equal(loose(case.batch, *case.raw), want)
    case.qw.data = case.qw.data.float()
    with pytest.raises(ValueError, match="query_weight"):
        case.step(case.batch, *case.raw)


def test_gains_and_sinks_that_autograd_follows():
    case = Case(heads=8, kv_heads=2, head_dim=64, pairs=32, norms=True, sinks=True, prefix=16, own=(3, 4))
    want = case.step(case.batch, *case.raw)
    grads = []
    for reference in (False, True):
        case.qw, case.kw, case.sinks = (torch.nn.Parameter(t.detach().clone()) for t in (case.qw, case.kw, case.sinks))
        step = case.make(case.cache, **(dict(reference=True) if reference else {}))
        before = dict(FALLBACKS)
        step(case.batch, *case.raw).float().square().sum().backward()
        assert reference or FALLBACKS != before
        grads.append([t.grad for t in (case.qw, case.kw, case.sinks)])
        if not reference:
            with torch.no_grad():   # nothing follows: the kernels, and the same result
                assert torch.equal(step(case.batch, *case.raw), want)
    assert all(torch.equal(a, b) and a.abs().max() > 0 for a, b in zip(*grads))


def test_a_mode_that_follows_a_call_sees_its_operations():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Names(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.add(func.name())
            return func(*args, **(kwargs or {}))

    case = Case(heads=8, kv_heads=2, head_dim=64, prefix=16, own=(3, 4))
    want = case.step(case.batch, *case.raw)
    with Names() as mode:
        mode.seen = set()
        got = case.step(case.batch, *case.raw)
    assert "aten::_softmax" in mode.seen
    assert (got.float() - want.float()).abs().max() <= 4 * HALF * want.float().abs().max()


def test_gradients_go_to_a_steps_own_rows():
    """Against the Core chain's, whose gradients are tested against the formula: the same chain."""
    case = Case(heads=8, kv_heads=2, head_dim=64, prefix=16, own=(3, 4), tokens=(2, 1))
    grads = []
    for step in (case.step, case.make(case.cache, reference=True)):
        raw = [t.clone().requires_grad_() for t in case.raw]
        step(case.batch, *raw).float().square().sum().backward()
        grads.append([t.grad for t in raw])
    assert all(torch.equal(a, b) and a.abs().max() > 0 for a, b in zip(*grads))
    assert not case.cache.keys.requires_grad


def test_what_cannot_be_captured_is_refused():
    case = Case(heads=8, kv_heads=2, head_dim=64, prefix=16, own=(3, 4))
    cache = case.cache
    refused = []
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: cache.open(3), lambda: cache.fork(case.chosen[0]), lambda: cache.free(case.chosen[0]),
                     lambda: cache.truncate(case.chosen[0], 1), cache.compact, lambda: cache.resize(500),
                     lambda: cache.batch(case.chosen), lambda: cache.reserve(case.chosen[0], 60)):
            try:
                call()
            except ValueError as error:
                refused.append("captured" in str(error))
        torch.zeros(1, device="cuda")
    assert refused == [True] * 8


def test_another_stream():
    case = Case(heads=32, kv_heads=8, head_dim=128, pairs=64, norms=True, page_rows=64, prefix=1024, own=(3, 70, 9))
    want = case.step(case.batch, *case.raw)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [case.step(case.batch, *case.raw) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(g, want) for g in got)


def test_two_threads_with_a_cache_each():
    made = [Case(heads=16, kv_heads=4, head_dim=128, pairs=64, page_rows=32, prefix=640, own=(3, 70 + i, 9), seed=i)
            for i in range(2)]
    want = [case.step(case.batch, *case.raw) for case in made]
    got: list = [[], []]
    torch.cuda.synchronize()

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(made[i].step(made[i].batch, *made[i].raw))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for mine, all_of in zip(want, got):
        assert len(all_of) == 20 and all(torch.equal(g, mine) for g in all_of)


def test_a_pool_that_grows_and_many_forks():
    """More children than one launch takes, then a pool of another size, then a step of them all."""
    case = Case(heads=8, kv_heads=2, head_dim=64, page_rows=16, prefix=0, own=(45,))
    parent, cache = case.chosen[0], case.cache
    wanted = cache.keys[1, cache.pages_of(parent)[2], :, :13].clone()
    grown = PagedKVCache.empty(2, 400, 16, 2, 64, device="cuda", sequences=300, rows=100)
    assert grown.open(45) == 0
    for mine, theirs in ((grown.keys, cache.keys), (grown.values, cache.values)):
        mine[:, grown.pages_of(0)] = theirs[:, cache.pages_of(parent)]
    kids = grown.fork(0, 270)
    assert all(torch.equal(grown.keys[1, grown.pages_of(kid)[2], :, :13], wanted) for kid in (kids[0], *kids[127:131], kids[-1]))
    step = case.make(grown)
    batch = grown.batch(kids)
    raw = [case.normal(270, n * 64) for n in (8, 2, 2)]
    want = step(batch, *raw)
    grown.resize(600)
    assert torch.equal(step(grown.batch(kids), *raw), want)
    few = step(grown.batch(kids[:5]), *(t[:5] for t in raw))
    grown.free(kids[5:])
    assert grown.compact() == 8
    grown.resize(8)
    assert torch.equal(step(grown.batch(kids[:5]), *(t[:5] for t in raw)), few)


def test_pools_past_32_bits():
    """Pages whose elements lie past 2^31 of their pool, and past 2^32 bytes."""
    kv_heads, head_dim, size = 8, 128, 256
    pages = (1 << 31) // (kv_heads * head_dim * size) + 60
    pool = torch.empty((1, pages, kv_heads, size, head_dim), dtype=torch.bfloat16, device="cuda")
    cache = PagedKVCache(pool, torch.empty_like(pool), sequences=4, rows=2048)
    gen = torch.Generator(device="cuda").manual_seed(1)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda").bfloat16()  # noqa: E731
    tables = np.full((4, 8), -1, dtype=np.int32)
    tables[0, :4], tables[1, :3], tables[1, 3] = [pages - 1, 2, pages - 3, pages - 5], [pages - 1, 2, pages - 3], pages - 2
    for page in [pages - 1, 2, pages - 3, pages - 5, pages - 2]:
        for p in (cache.keys, cache.values):
            p[0, page] = normal(kv_heads, size, head_dim)
    cache = PagedKVCache(cache.keys, cache.values, tables=tables, lengths=np.array([800, 900, 0, 0]), opened=[0, 1])
    batch = cache.batch([0, 1])
    assert batch.prefix == 768
    step = BatchAttentionStep(cache, layer=0, heads=32, kv_heads=8, head_dim=128, scale=128 ** -0.5, dtype=torch.bfloat16)
    raw = [normal(2, n * 128) for n in (32, 8, 8)]
    out = step(batch, *raw)
    # The same rows in a pool of their own.
    names = {page: i for i, page in enumerate([pages - 1, 2, pages - 3, pages - 5, pages - 2])}
    small = [torch.stack([p[0, page] for page in names])[None] for p in (cache.keys, cache.values)]
    near = np.array([[names.get(page, -1) for page in row] for row in tables])
    twin = PagedKVCache(*small, tables=near, lengths=np.array([800, 900, 0, 0]), opened=[0, 1])
    other = BatchAttentionStep(twin, layer=0, heads=32, kv_heads=8, head_dim=128, scale=128 ** -0.5, dtype=torch.bfloat16)
    assert torch.equal(other(twin.batch([0, 1]), *raw), out)
    kids = cache.fork(1, 2)   # the last page copied, to the front of the pool
    for kid in kids:
        assert torch.equal(cache.keys[0, cache.pages_of(kid)[3], :, :132], cache.keys[0, pages - 2, :, :132])
    cache.free([0, *kids])
    want = cache.keys[0, [pages - 1, 2, pages - 3]].clone()
    assert cache.compact() == 4
    assert torch.equal(cache.keys[0, cache.pages_of(1)[:3]], want)
    assert cache.tables[1, :4].tolist() == cache.pages_of(1)


# The cache's own kernels ----------------------------------------------------------------------


@pytest.mark.parametrize("seed", range(4))
def test_any_order_of_calls_keeps_every_sequence(seed):
    rng = np.random.default_rng(seed)
    cache = PagedKVCache.empty(int(rng.integers(1, 4)), int(rng.integers(8, 30)), 16, 2, 16, device="cuda",
                               sequences=int(rng.integers(2, 9)), rows=100)
    random_calls(cache, PagedModel(), rng, 60, check_every=5)


def test_a_cache_of_many_pages_is_the_hosts():
    """More entries, children and moves than one launch takes: the tables, the lengths and the
    pages of the same calls on the CPU."""
    caches = [PagedKVCache.empty(2, 900, 16, 2, 8, device=device, sequences=400, rows=3200) for device in ("cuda", "cpu")]
    gen = torch.Generator().manual_seed(5)
    first = torch.randn(caches[1].keys.shape, generator=gen).bfloat16()
    for cache in caches:
        for pool in (cache.keys, cache.values):
            pool.copy_(first)
    rng = np.random.default_rng(1)

    def same(call):
        got = [call(cache) for cache in caches]
        assert got[0] == got[1]
        device, host = caches
        assert torch.equal(device.tables.cpu(), host.tables) and torch.equal(device.lengths.cpu(), host.lengths)
        assert torch.equal(device.keys.cpu(), host.keys) and torch.equal(device.values.cpu(), host.values)
        for name in ("_tables", "_rows", "_held", "_refs", "_generation", "_open"):
            assert np.array_equal(getattr(device, name), getattr(host, name)), name
        assert device._epoch == host._epoch
        return got[0]

    assert same(lambda c: c.open(2500)) == 0 and same(lambda c: c.open(3200)) == 1
    kids = same(lambda c: c.fork(0, 300))
    gone = [int(s) for s in rng.permutation(kids)[:170]]
    same(lambda c: c.free([1, *gone]))
    for rows in (0, 1, 16, 17, 2080):
        same(lambda c: c.open(rows))
    same(lambda c: c.free(0))
    assert same(lambda c: c.compact()) == caches[0].pages - caches[0].free_pages
    same(lambda c: c.fork(kids[-1] if kids[-1] not in gone else [s for s in kids if s not in gone][0], 2, share=False))
    same(lambda c: c.resize(1000))
    same(lambda c: c.free([s for s in kids if s not in gone][:100]))
    same(lambda c: c.compact())
    for call in (lambda c: c.open(3201), lambda c: c.open(3200) and c.open(3200) and c.open(3200) and c.open(3200)):
        errors = []
        for cache in caches:
            with pytest.raises(ValueError) as refused:
                for _ in range(9):
                    call(cache)
            errors.append(str(refused.value).rsplit(": ", 1)[1].split(" (code")[0])
        assert errors[0] == errors[1]
    same(lambda c: c.compact())


@pytest.mark.parametrize("dtype,head_dim", [(torch.bfloat16, 8), (torch.bfloat16, 128), (torch.float32, 24)])
def test_copies_of_many_pages(dtype, head_dim):
    """More moves than one launch takes, whole and partial rows, and the tables renamed."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    shape = (3, 700, 3, 16, head_dim)
    keys, values = (torch.randn(shape, generator=gen, device="cuda").to(dtype) for _ in range(2))
    before = keys.clone(), values.clone()
    moves = [(350 + i, 349 - i, 1 + i % 16) for i in range(340)]
    tables = torch.randint(-1, 700, (40, 33), generator=gen, device="cuda", dtype=torch.int32)
    old = tables.clone()
    ops.pages_copy(keys, values, moves, tables=tables)
    names = torch.arange(-1, 700, device="cuda", dtype=torch.int32)
    for source, target, rows in moves:
        names[source + 1] = target
        for was, now in zip(before, (keys, values)):
            was[:, target, :, :rows] = was[:, source, :, :rows]
    assert torch.equal(keys, before[0]) and torch.equal(values, before[1])
    assert torch.equal(tables, names[old.long() + 1])


def test_ops_refuse():
    case = Case(heads=8, kv_heads=2, head_dim=128, pairs=64, prefix=32, own=(3, 4))
    cache, batch, tiles = case.cache, case.batch, case.batch.tiles(4)
    q = case.step.project(batch, *case.raw)
    keys, values = cache.keys[1], cache.values[1]
    base = dict(prefix=32, own_rows=5, scale=1.0)
    calls = [
        lambda: ops.attention_batch(q.half(), keys, values, cache.tables, cache.lengths, batch.token_map, tiles, **base),
        lambda: ops.attention_batch(q[:, ::2], keys, values, cache.tables, cache.lengths, batch.token_map, tiles, **base),
        lambda: ops.attention_batch(q, keys.float(), values, cache.tables, cache.lengths, batch.token_map, tiles, **base),
        lambda: ops.attention_batch(q, keys, values, cache.tables.long(), cache.lengths, batch.token_map, tiles, **base),
        lambda: ops.attention_batch(q, keys, values, cache.tables, cache.lengths[:2], batch.token_map, tiles, **base),
        lambda: ops.attention_batch(q, keys, values, cache.tables, cache.lengths, batch.token_map[:1], tiles, **base),
        lambda: ops.attention_batch(q, keys, values, cache.tables, cache.lengths, batch.token_map, tiles[:, :2], **base),
        lambda: ops.attention_batch(q, keys, values, cache.tables, cache.lengths, batch.token_map, tiles.cpu(), **base),
        lambda: ops.attention_batch(q, keys, values, cache.tables, cache.lengths, batch.token_map, tiles,
                                    prefix_sequence=cache.tables.shape[0], **base),
        lambda: ops.attention_batch(q, keys, values, cache.tables, cache.lengths, batch.token_map, tiles, prefix=-1,
                                    own_rows=5, scale=1.0),
        lambda: ops.attention_batch(q, keys, values, cache.tables, cache.lengths, batch.token_map, tiles, prefix=32,
                                    own_rows=5, scale=0.0),
        lambda: ops.attention_batch(q, keys, values, cache.tables, cache.lengths, batch.token_map, tiles,
                                    sinks=torch.zeros(7, device="cuda").bfloat16(), **base),
        lambda: ops.attention_batch_project(case.raw[0][:1], *case.raw[1:], None, None, None, keys, values,
                                            cache.tables, cache.lengths, batch.token_map, heads=8, eps=1e-6),
        lambda: ops.attention_batch_project(*case.raw, None, None, (case.cos, case.sin[:, :32]), keys, values,
                                            cache.tables, cache.lengths, batch.token_map, heads=8, eps=1e-6),
        lambda: ops.pages_copy(cache.keys[:, ::2], cache.values[:, ::2], [(0, 1, 1)]),
        lambda: ops.pages_copy(cache.keys, cache.values, [(0, cache.pages, 1)]),
        lambda: ops.pages_copy(cache.keys, cache.values, [(0, 1, 1), (2, 1, 1)] * 200),
        lambda: ops.pages_edit(cache.tables, cache.lengths, cache.pages, [(0, 0, 0, 1 << 40)]),
        lambda: ops.pages_edit(cache.tables, cache.lengths, cache.pages, [(0, 0, 0)]),
        lambda: ops.pages_advance(cache.lengths, batch.chosen, batch.rows[:1]),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    short = BatchAttentionStep(cache, layer=0, heads=8, kv_heads=2, head_dim=128, scale=1.0, dtype=torch.bfloat16,
                               rotary_pairs=64, angles=AngleTable(case.cos[:20], case.sin[:20]))
    with pytest.raises(ValueError, match="angle table"):
        short(batch, *case.raw)


# A run of them together -----------------------------------------------------------------------


def test_answers_sampled_from_one_prompt():
    """Two layers: a prompt taken in, forked, stepped, some answers freed, the pool compacted
    and the rest stepped on, against the same sequences with pages of their own and against the
    oracle; the angles an atlas that grows on the way."""
    heads, kv_heads, d, layers = 8, 2, 128, 2
    gen = torch.Generator(device="cuda").manual_seed(4)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda").bfloat16()  # noqa: E731
    gains = [(1 + 0.1 * normal(d).float()).bfloat16() for _ in range(2)]
    atlas = AngleAtlas(64, base=1e6, rows=64, device="cuda")

    def layered(share):
        cache = PagedKVCache.empty(layers, 90, 32, kv_heads, d, device="cuda", sequences=9, rows=400)
        steps = [BatchAttentionStep(cache, layer=i, heads=heads, kv_heads=kv_heads, head_dim=d, scale=d ** -0.5,
                                    dtype=torch.bfloat16, query_weight=gains[0], key_weight=gains[1],
                                    rotary_pairs=64, angles=atlas) for i in range(layers)]
        return cache, steps, share

    def advance(cache, steps, batch, raw):
        outs = [step(batch, *(t * (i + 1) for t in raw)) for i, step in enumerate(steps)]
        cache.advance(batch)
        return torch.stack(outs)

    worlds = [layered(True), layered(False)]
    prompt = [normal(150, n * d) for n in (heads, kv_heads, kv_heads)]
    first = []
    for cache, steps, _ in worlds:
        assert cache.open() == 0
        first.append(advance(cache, steps, cache.batch([0], tokens=150), prompt))
    assert torch.equal(*first)
    kids = [cache.fork(0, 5, share=share) for cache, _, share in worlds]
    assert kids[0] == kids[1] and worlds[0][0].free_pages > worlds[1][0].free_pages
    batches = [cache.batch(kids[0]) for cache, _, _ in worlds]
    assert batches[0].prefix == 128 and batches[1].prefix == 0
    close = lambda a, b: (a.float() - b.float()).abs().max() <= 4 * HALF * b.float().abs().max()  # noqa: E731
    for turn in range(40):
        if turn == 15:
            for cache, _, _ in worlds:
                cache.free([kids[0][1], 0])
                cache.compact()
            batches = [cache.batch([kids[0][i] for i in (4, 0, 2, 3)]) for cache, _, _ in worlds]
            assert batches[0].prefix == 128
        raw = [normal(batches[0].total, n * d) for n in (heads, kv_heads, kv_heads)]
        outs = [advance(cache, steps, batch, raw) for (cache, steps, _), batch in zip(worlds, batches)]
        assert close(*outs), turn
    cache = worlds[0][0]
    assert cache.rows(kids[0][0]) == 190 and atlas.rows >= 190
    table = atlas.table()
    queries = ops.attention_batch_project(
        *raw, *gains, (table.cos, table.sin), cache.keys[1], cache.values[1], cache.tables, cache.lengths,
        batches[0].token_map, heads=heads, eps=1e-6, wide_queries=True)
    got = worlds[0][1][1](batches[0], *raw)
    want, size = attend(wide(queries), wide(cache.keys[1]), wide(cache.values[1]), cache.tables.cpu().numpy(),
                        cache.lengths.cpu().numpy(), batches[0].token_map.cpu().numpy(), d ** -0.5)
    assert np.all(np.abs(wide(got) - want) <= HALF * np.abs(want) + (HALF + 2.0 ** -12) * size)


@pytest.mark.parametrize("tokens", [1, 3, 5])
def test_one_long_sequence_among_short_ones(tokens):
    """Pieces cut for what the sequences hold together, and for the longest alone where that is not known."""
    case = Case(heads=8, kv_heads=2, head_dim=64, pairs=32, page_rows=64, own=(9000, *(i % 41 for i in range(60))), tokens=tokens)
    context = case.check(np.arange(0, case.batch.total, 13))
    queries, group = case.wide_queries(), 4
    tiles = case.batch.tiles(group)
    assert case.batch.own_total(group) == sum(int(case.cache.rows(s)) + tokens for s in case.chosen)
    other = ops.attention_batch(queries, case.cache.keys[1], case.cache.values[1], case.cache.tables, case.cache.lengths,
                                case.batch.token_map, tiles, prefix=0, own_rows=9000 + tokens, scale=case.scale)
    case.check_context(other, queries, case.cache.lengths.cpu().numpy(), np.arange(0, case.batch.total, 13))
    assert (other.float() - context.float()).abs().max() <= 4 * HALF * context.float().abs().max()


def test_another_device_than_the_current_one_is_refused(monkeypatch):
    """Before anything is launched or counted: the tensors' device would not be the one that runs."""
    case = Case(heads=8, kv_heads=2, head_dim=128, pairs=64, norms=True, prefix=64, own=(3, 4))
    cache, tables = case.cache, case.cache.tables.clone()
    want = case.step(case.batch, *case.raw)
    held, rows = cache.free_pages, cache.rows(case.chosen[0])
    with monkeypatch.context() as patch:
        patch.setattr(ops, "_current_device", lambda: 1)
        for call in (lambda: case.step(case.batch, *case.raw), lambda: case.step.project(case.batch, *case.raw),
                     lambda: cache.open(20), lambda: cache.fork(case.chosen[0]), lambda: cache.free(case.chosen[0]),
                     cache.compact, lambda: cache.advance(case.batch), lambda: cache.reserve(case.chosen[0], 99),
                     lambda: cache.truncate(case.chosen[0], 1), lambda: cache.resize(500),
                     lambda: cache.fork(case.chosen[0], share=False), lambda: ops.pages_advance(cache.lengths, case.batch.chosen, case.batch.rows),
                     case.wide_queries, lambda: ops.pages_copy(cache.keys, cache.values, [(0, 1, 1)]),
                     lambda: ops.pages_edit(cache.tables, cache.lengths, cache.pages, [(0, 0, 0, 1)])):
            with pytest.raises(ValueError, match="is current"):
                call()
    assert cache.free_pages == held and cache.rows(case.chosen[0]) == rows and torch.equal(cache.tables, tables)
    assert torch.equal(case.step(case.batch, *case.raw), want)
