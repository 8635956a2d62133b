"""The cache of pages and the batch step on the CPU: what the tables say after every kind of
call, refusals, and the Core chain against the float64 oracle."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mlx_omnia_amd.kernels.attention import (BatchAttentionStep, DefaultBatchAttentionStep, PagedKVCache,
                                             batch_step_applies)
from mlx_omnia_amd.kernels.qkv_rope import AngleAtlas, AngleTable
from mlx_omnia_amd.runtime import ops
from oracle.batch_attention import attend, turned
from paged_model import PagedModel, check_against, random_calls


def small(pages=12, page_rows=16, sequences=6, rows=96, layers=2, kv_heads=2, head_dim=8):
    return PagedKVCache.empty(layers, pages, page_rows, kv_heads, head_dim, sequences=sequences, rows=rows)


def test_pages_are_handed_out_lowest_first():
    cache = small()
    a, b = cache.open(40), cache.open(1)
    assert (a, b) == (0, 1) and cache.pages_of(a) == [0, 1, 2] and cache.pages_of(b) == [3]
    cache.free(a)
    assert cache.open(17) == 0 and cache.pages_of(0) == [0, 1]
    assert cache.tables[0].tolist() == [0, 1, -1, -1, -1, -1] and cache.lengths.tolist() == [17, 1, 0, 0, 0, 0]
    assert cache.free_pages == 9


def test_fork_shares_full_pages_and_copies_the_rest():
    cache = small()
    cache.keys.copy_(torch.arange(cache.keys.numel()).reshape(cache.keys.shape))
    parent = cache.open(40)
    before = cache.keys.clone()
    one, two = cache.fork(parent, 2)
    assert cache.pages_of(one) == [0, 1, 3] and cache.pages_of(two) == [0, 1, 4]
    assert torch.equal(cache.keys[:, 3, :, :8], before[:, 2, :, :8])
    assert torch.equal(cache.keys[:, 3, :, 8:], before[:, 3, :, 8:])   # rows past the last, left alone
    cache.free([parent, one])
    assert cache.pages_of(two) == [0, 1, 4] and cache.free_pages == 9
    (whole,) = cache.fork(two, 1, share=False)
    assert cache.pages_of(whole) == [2, 3, 5] and cache.rows(whole) == 40


@pytest.mark.parametrize("rows", [0, 16, 32])
def test_fork_at_a_page_end_copies_nothing(rows):
    cache = small()
    parent = cache.open(rows)
    cache.reserve(parent, rows + 20)
    (kid,) = cache.fork(parent)
    assert cache.pages_of(kid) == cache.pages_of(parent)[: rows // 16] and cache.rows(kid) == rows


def test_a_shared_page_is_copied_before_it_is_written():
    cache = small()
    parent = cache.open(32)
    kids = cache.fork(parent, 2)
    for s in (parent, *kids):
        cache.truncate(s, 20)
    assert cache.pages_of(parent) == [0, 1] == cache.pages_of(kids[0])
    batch = cache.batch([parent, *kids])
    assert batch.prefix == 16
    cache.ready(batch)
    # The last of the three keeps the page; the others have copies.
    assert [cache.pages_of(s) for s in (parent, *kids)] == [[0, 2], [0, 3], [0, 1]]
    assert cache.ready(batch) == 21 and cache.pages_of(parent) == [0, 2]


def test_a_page_that_others_keep_is_copied_for_all():
    cache = small()
    parent = cache.open(32)
    kids = cache.fork(parent, 2)
    cache.truncate(kids[0], 17)
    cache.ready(cache.batch([kids[0]]))
    assert cache.pages_of(kids[0]) == [0, 2] and cache.pages_of(kids[1]) == [0, 1] == cache.pages_of(parent)


def test_compact_and_resize():
    cache = small()
    cache.keys.copy_(torch.arange(cache.keys.numel()).reshape(cache.keys.shape))
    first, second, third = cache.open(30), cache.open(20), cache.open(16)
    held = cache.keys[:, [2, 3, 4]].clone()
    cache.free(first)
    with pytest.raises(ValueError, match="too few"):
        cache.resize(3)
    assert cache.compact() == 3
    assert cache.pages_of(second) == [2, 0] and cache.pages_of(third) == [1]
    assert cache.tables[second, :3].tolist() == [2, 0, -1] and cache.tables[third, 0] == 1
    assert torch.equal(cache.keys[:, [2, 0, 1]], held)
    assert cache.compact() == 3 and cache.pages_of(second) == [2, 0]
    cache.resize(3)
    assert cache.pages == 3 and cache.free_pages == 0 and torch.equal(cache.keys[:, [2, 0, 1]], held)
    cache.resize(5)
    assert cache.free_pages == 2 and torch.equal(cache.keys[:, [2, 0, 1]], held)


def test_batches_find_what_their_sequences_share():
    cache = small(pages=20)
    parent = cache.open(50)
    kids = cache.fork(parent, 3)
    other = cache.open(33)
    assert cache.batch(kids).prefix == 48 and cache.batch([parent]).prefix == 0
    assert cache.batch([*kids, other]).prefix == 0
    cache.truncate(kids[1], 40)
    assert cache.batch(kids).prefix == 32
    batch = cache.batch([kids[0], kids[2]], tokens=[3, 1])
    assert batch.token_map.tolist() == [[kids[0], 0], [kids[0], 1], [kids[0], 2], [kids[2], 0]]
    assert batch.tiles(50).tolist() == [[0, 128, kids[0], 0], [128, 150, kids[0], 2], [150, 200, kids[2], 0]]


def test_children_in_the_slots_that_are_left():
    cache = small(pages=20, sequences=7)
    for _ in range(6):
        cache.open(3)
    cache.free([4, 1, 3])
    assert cache.fork(0, 3) == [1, 3, 4]
    assert [cache.pages_of(s) for s in (1, 3, 4)] == [[1], [3], [4]] and cache.pages_of(5) == [5]
    assert cache.tables[:, 0].tolist() == [0, 1, 2, 3, 4, 5, -1] and cache.lengths.tolist() == [3] * 6 + [0]
    assert cache.open() == 6 and cache.fork(0, 0) == []


def test_full_pools_and_tables_leave_everything_as_it_was():
    cache = small(pages=4, sequences=3, rows=64)
    a = cache.open(40)
    state = lambda: (cache.tables.clone(), cache.lengths.clone(), cache.free_pages)  # noqa: E731
    before = state()
    for call, text in ((lambda: cache.open(40), "2 more|3 more pages"), (lambda: cache.open(65), "at most 64"),
                       (lambda: cache.reserve(a, 65), "at most 64"), (lambda: cache.fork(a, 2), "2 more pages"),
                       (lambda: cache.fork(a, 3), "3 more sequences"), (lambda: cache.fork(a, 1, share=False), "pages"),
                       (lambda: cache.ready(cache.batch([a], tokens=30)), "at most 64")):
        with pytest.raises(ValueError, match=text):
            call()
        after = state()
        assert torch.equal(before[0], after[0]) and torch.equal(before[1], after[1]) and before[2] == after[2]


def test_refusals():
    cache = small()
    a, b = cache.open(20), cache.open(20)
    for call in (lambda: cache.open(-1), lambda: cache.free([a, a]), lambda: cache.free(5), lambda: cache.fork(5),
                 lambda: cache.fork(a, -1), lambda: cache.truncate(a, 21), lambda: cache.truncate(a, -1),
                 lambda: cache.batch([]), lambda: cache.batch([a, a]), lambda: cache.batch([a, 5]),
                 lambda: cache.batch([a, b], tokens=[1]), lambda: cache.batch([a], tokens=0),
                 lambda: cache.batch([-1]), lambda: cache.rows(-1)):
        with pytest.raises(ValueError):
            call()
    batch = cache.batch([a, b])
    with pytest.raises(ValueError, match="another cache"):
        small().advance(batch)
    with pytest.raises(ValueError, match="more steps"):
        cache.account(batch, 13)
    with pytest.raises(ValueError, match="at least once"):
        cache.prepare_capture(batch, 0)
    cache.free(b)
    for call in (lambda: cache.ready(batch), lambda: cache.advance(batch)):
        with pytest.raises(ValueError, match="freed or truncated"):
            call()
    cache.open()
    with pytest.raises(ValueError, match="freed or truncated"):   # the slot is another sequence now
        cache.advance(batch)


@pytest.mark.parametrize("change", [
    dict(tables=np.full((2, 2), -1)), dict(tables=np.zeros((2, 2), int), lengths=np.zeros(2, int)), dict(sequences=2),
    dict(tables=np.array([[5, -1]]), lengths=np.array([1]), opened=[0]),
    dict(tables=np.array([[-1, 1]]), lengths=np.array([1]), opened=[0]),
    dict(tables=np.array([[1, 1]]), lengths=np.array([1]), opened=[0]),
    dict(tables=np.array([[1, -1]]), lengths=np.array([17]), opened=[0]),
    dict(tables=np.array([[1, -1]]), lengths=np.array([3]), opened=[]),
    dict(tables=np.array([[1, -2]]), lengths=np.array([3]), opened=[0]), dict(sequences=0, rows=3),
    dict(sequences=2, rows=16, opened=[0]), dict(tables=np.array([[1, -1]]), lengths=np.array([3]), opened=[-1]),
    dict(tables=np.array([[1, -1]]), lengths=np.array([3]), opened=[0, 1]),
    dict(tables=np.array([[1, -1]]), lengths=np.array([3]), opened=[0, 0]),
    # a page that both sequences would write next, one shared and one not yet reached
    dict(tables=np.array([[0, 1], [2, 1]]), lengths=np.array([16, 16]), opened=[0, 1]),
    dict(tables=np.array([[0, 1], [2, 1]]), lengths=np.array([16, 20]), opened=[0, 1])])
def test_tables_that_do_not_hold_together_are_refused(change):
    pool = torch.zeros((1, 4, 2, 16, 8))
    with pytest.raises(ValueError):
        PagedKVCache(pool, pool.clone(), **change)


@pytest.mark.parametrize("shape", [(1, 4, 2, 24, 8), (1, 4, 2, 512, 8), (1, 4, 2, 16, 12), (4, 2, 16, 8), (1, 0, 2, 16, 8)])
def test_pools_of_other_shapes_are_refused(shape):
    pool = torch.zeros(shape)
    with pytest.raises(ValueError):
        PagedKVCache(pool, pool.clone(), sequences=2, rows=16)


@pytest.mark.parametrize("seed", range(6))
def test_any_order_of_calls_keeps_every_sequence(seed):
    """Rows are numbered as they are written; after each of 120 random calls every open
    sequence holds the rows that a list a sequence says it holds."""
    rng = np.random.default_rng(seed)
    cache = small(pages=int(rng.integers(8, 30)), page_rows=16, sequences=int(rng.integers(2, 9)), rows=100)
    random_calls(cache, PagedModel(), rng, 120)


def test_whole_numbers_of_numpy():
    cache = small()
    a, b = cache.open(np.int64(3)), cache.open(5)
    batch = cache.batch(np.array([a, b]), tokens=np.int32(2))
    cache.ready(batch)
    cache.advance(batch)
    assert cache.rows(np.int64(a)) == 5
    cache.free(np.int64(a))
    cache.free(np.array([b]))
    assert cache.free_pages == cache.pages


def test_a_cache_is_taken_up_as_it_was_left():
    rng = np.random.default_rng(3)
    cache, model = small(pages=20), PagedModel()
    random_calls(cache, model, rng, 60)
    again = PagedKVCache(cache.keys.clone(), cache.values.clone(), tables=cache.tables.numpy(),
                         lengths=cache.lengths.numpy(), opened=list(model.rows))
    check_against(again, model)
    random_calls(again, model, rng, 60)


# The Core chain -----------------------------------------------------------------------------


def filled(rng, cache):
    for pool in (cache.keys, cache.values):
        pool.copy_(torch.from_numpy(rng.standard_normal(tuple(pool.shape)).astype(np.float32)))


@pytest.mark.parametrize("heads,kv_heads,head_dim,pairs,norms,sinks,tokens", [
    (4, 2, 8, 4, True, False, 1), (6, 2, 8, 0, False, True, [3, 1, 5]), (3, 3, 16, 8, True, True, [1, 17, 2])])
def test_core_chain_against_the_oracle(heads, kv_heads, head_dim, pairs, norms, sinks, tokens):
    rng = np.random.default_rng(heads)
    cache = PagedKVCache.empty(2, 24, 16, kv_heads, head_dim, sequences=5, rows=90, dtype=torch.float32)
    filled(rng, cache)
    parent = cache.open(37)
    chosen = [*cache.fork(parent, 2), cache.open(0)] if heads == 6 else cache.fork(parent, 3)
    batch = cache.batch(chosen, tokens=tokens)
    raw = [rng.standard_normal((batch.total, n * head_dim)) for n in (heads, kv_heads, kv_heads)]
    gains = [1 + 0.1 * rng.standard_normal(head_dim) for _ in range(2)] if norms else [None, None]
    cos, sin = (np.cos(rng.uniform(0, 6, (90, pairs))), np.sin(rng.uniform(0, 6, (90, pairs))))
    logits = rng.standard_normal(heads) if sinks else None
    tensor = lambda a: None if a is None else torch.from_numpy(np.asarray(a)).float()  # noqa: E731
    step = BatchAttentionStep(
        cache, layer=1, heads=heads, kv_heads=kv_heads, head_dim=head_dim, scale=0.3, dtype=torch.float32,
        query_weight=tensor(gains[0]), key_weight=tensor(gains[1]), eps=1e-6, rotary_pairs=pairs, mscale=1.25,
        angles=AngleTable(tensor(cos), tensor(sin)) if pairs else None, sinks=tensor(logits))
    assert isinstance(step.strategy, DefaultBatchAttentionStep)
    untouched = cache.keys[0].clone()
    context = step(batch, *(tensor(a) for a in raw))
    assert torch.equal(cache.keys[0], untouched)
    token_map, lengths = batch.token_map.numpy(), cache.lengths.numpy()
    f32 = np.float32(1) * 2.0 ** -18   # a few dozen operations of half a step of 2^-24 each
    queries = np.zeros((batch.total, heads, head_dim))
    for t, (s, j) in enumerate(token_map):
        p = lengths[s] + j
        angles = (cos[p].astype(np.float32), sin[p].astype(np.float32)) if pairs else (None, None)
        f = lambda a: None if a is None else np.asarray(a, dtype=np.float32)  # noqa: E731
        queries[t] = turned(f(raw[0][t]).reshape(heads, -1), f(gains[0]), *angles, 1e-6, 1.25)
        key = turned(f(raw[1][t]).reshape(kv_heads, -1), f(gains[1]), *angles, 1e-6, 1.25)
        page = cache.tables[s, p // 16]
        assert np.abs(cache.keys[1, page, :, p % 16].numpy() - key).max() <= f32 * (1 + np.abs(key).max())
        assert np.array_equal(cache.values[1, page, :, p % 16].numpy(), f(raw[2][t]).reshape(kv_heads, -1))
    want, size = attend(queries, cache.keys[1].numpy(), cache.values[1].numpy(), cache.tables.numpy(), lengths,
                        token_map, 0.3, f(logits) if sinks else None)
    assert np.all(np.abs(context.numpy() - want) <= 2.0 ** -14 * (size + 1e-3))


def test_core_chain_keeps_a_later_tokens_infinity_from_an_earlier_one():
    cache = PagedKVCache.empty(1, 4, 16, 1, 8, sequences=1, rows=40, dtype=torch.float32)
    cache.open(5)
    batch = cache.batch([0], tokens=3)
    step = BatchAttentionStep(cache, layer=0, heads=1, kv_heads=1, head_dim=8, scale=1.0, dtype=torch.float32)
    v = torch.ones(3, 8)
    v[2, 3] = float("inf")
    out = step(batch, torch.ones(3, 8), torch.ones(3, 8), v)
    assert torch.isfinite(out[:2]).all() and torch.isinf(out[2, 0, 3]) and torch.isfinite(out[2, 0, :3]).all()


def test_gradients_of_a_steps_own_rows():
    """Against the formula in 64 bits and its central differences; earlier rows are constants, and
    the pool keeps no graph. The step's operations are some thousand fp32 ones a number, none of
    which cancels by more than the 2^6 that the sums of its terms' sizes allow: 2^-24 2^6 2^5."""
    gen = torch.Generator().manual_seed(2)
    heads, kv, d, scale = 4, 2, 8, 0.4
    cache = PagedKVCache.empty(2, 9, 16, kv, d, sequences=3, rows=48, dtype=torch.float32)
    for pool in (cache.keys, cache.values):
        pool.copy_(torch.randn(pool.shape, generator=gen))
    chosen = [cache.open(21)]
    chosen += cache.fork(chosen[0])
    counts = [3, 1]
    batch = cache.batch(chosen, tokens=counts)
    step = BatchAttentionStep(cache, layer=1, heads=heads, kv_heads=kv, head_dim=d, scale=scale, dtype=torch.float32)
    old = [[torch.stack([pool[1, cache.tables[s, r // 16], :, r % 16] for r in range(21)]).double() for s in chosen]
           for pool in (cache.keys, cache.values)]
    raw = [torch.randn(batch.total, n * d, generator=gen) for n in (heads, kv, kv)]
    weight = torch.randn(batch.total, heads, d, generator=gen)

    def formula(q, k, v):
        total, at = 0.0, 0
        for i, n in enumerate(counts):
            for t in range(n):
                for h in range(heads):
                    keys, values = (torch.cat([o[i][:, h // 2], new[at : at + t + 1].unflatten(1, (kv, d))[:, h // 2]])
                                    for o, new in zip(old, (k, v)))
                    p = torch.softmax(keys @ q[at + t].unflatten(0, (heads, d))[h] * scale, dim=0)
                    total = total + (p @ values) @ weight[at + t, h].double()
            at += n
        return total

    mine = [t.clone().requires_grad_() for t in raw]
    (step(batch, *mine) * weight).sum().backward()
    exact = [t.double().requires_grad_() for t in raw]
    formula(*exact).backward()
    for got, want in zip(mine, exact):
        assert (got.grad.double() - want.grad).abs().max() <= 2.0 ** -13 * want.grad.abs().max()
    along = [torch.randn(t.shape, generator=gen, dtype=torch.float64) for t in raw]
    h = 1e-5   # the differences' own error: h^2 of a third derivative of some hundreds, 2^-52 of some tens / h
    ends = [formula(*(t.double() + sign * h * a for t, a in zip(raw, along))) for sign in (1, -1)]
    slope = sum((t.grad * a).sum() for t, a in zip(exact, along))
    assert abs((ends[0] - ends[1]) / (2 * h) - slope) <= 1e-6 * (1 + abs(slope))
    assert not cache.keys.requires_grad and not cache.values.requires_grad
    assert torch.equal(step(batch, *raw), step(batch, *mine).detach())


def test_step_declarations():
    cache = small(head_dim=64)
    kind = dict(scale=1.0, dtype=torch.bfloat16)
    for bad in (dict(layer=2, heads=4, kv_heads=2, head_dim=64), dict(layer=0, heads=5, kv_heads=2, head_dim=64),
                dict(layer=0, heads=4, kv_heads=4, head_dim=64), dict(layer=0, heads=4, kv_heads=2, head_dim=128),
                dict(layer=0, heads=4, kv_heads=2, head_dim=64, rotary_pairs=32)):
        with pytest.raises(ValueError):
            BatchAttentionStep(cache, **bad, **kind)
    step = BatchAttentionStep(cache, layer=0, heads=4, kv_heads=2, head_dim=64, rotary_pairs=32, base=1e4, **kind)
    assert isinstance(step.strategy, DefaultBatchAttentionStep) and isinstance(step.strategy.angles, AngleAtlas)
    cache.open(3)
    batch = cache.batch([0])
    good = [torch.zeros(1, 256), torch.zeros(1, 128), torch.zeros(1, 128)]
    assert step(batch, *good).shape == (1, 4, 64)
    for i in range(3):
        bad = list(good)
        bad[i] = torch.zeros(2, bad[i].shape[1])
        with pytest.raises(ValueError, match="tokens"):
            step(batch, *bad)
    with pytest.raises(ValueError, match="captured"):
        step.prepare_capture(batch, 3)


@pytest.mark.parametrize("heads,kv_heads,head_dim,pairs,served", [
    (32, 8, 128, 64, True), (64, 8, 64, 32, True), (5, 5, 128, 0, True), (10, 2, 64, 8, True), (32, 8, 96, 32, False),
    (32, 8, 128, 60, False), (32, 8, 64, 40, False), (32, 5, 64, 32, False), (8192, 8, 64, 32, False)])
def test_what_the_kernels_serve(heads, kv_heads, head_dim, pairs, served):
    assert batch_step_applies(heads, kv_heads, head_dim, pairs) == served


# What the library refuses, before it looks for a device ---------------------------------------


def test_workspace_bytes():
    from mlx_omnia_amd.runtime import library
    nbytes = library().omnia_attention_batch_workspace_bytes
    assert nbytes(0, 32, 8, 128, 0, 1, 0, 0) == 0
    for total in (0, 1, 64 * 700, 1 << 50):
        assert nbytes(64, 32, 8, 128, 8192, 700, total, 64) % (64 * 32 * 130 * 4) == 0
    for bad in ((1, 32, 8, 96, 0, 1, 0, 1), (1, 32, 5, 128, 0, 1, 0, 1), (1, 32, 8, 128, -1, 1, 0, 1),
                (1, 32, 8, 128, 0, 1 << 30, 0, 1), (1 << 28, 32, 8, 128, 0, 1, 0, 1), (1, 8192, 8, 128, 0, 1, 0, 1),
                (1, 32, 8, 128, 0, 1, -1, 1)):
        assert nbytes(*bad) < 0


def _copy(moves, *, layers=1, pages=8, heads=2, rows=16, dim=64, tables=None, entries=0):
    from mlx_omnia_amd.runtime import library, loader
    flat = ops._int_lines(moves, 3, "moves")
    rc = library().omnia_pages_copy(4096, 8192, layers, pages, heads, rows, dim, flat.buffer_info()[0], len(moves), tables,
                                    entries, None)
    return rc, loader.last_error()


@pytest.mark.parametrize("moves,text,more", [
    ([(0, 8, 1)], "no such page", {}), ([(-1, 2, 1)], "no such page", {}), ([(1 << 30, 2, 1)], "no such page", {}),
    ([(0, 1, 0)], "rows outside", {}), ([(0, 1, 17)], "rows outside", {}), ([(0, 1, 4), (2, 1, 4)], "two moves", {}),
    ([(0, 1, 4), (1, 2, 4)], "both read", {}), ([(3, 3, 4)], "both read", {}),
    ([(4, 0, 4), (3, 1, 4)], "sorted", dict(tables=4096, entries=4)), ([(0, 1, 1)], "bad page", dict(dim=60)),
    ([(0, 1, 1)], "bad pool", dict(layers=0)), ([(0, 1, 1)] * 129, "more moves", {})])
def test_pages_copy_refuses(moves, text, more):
    rc, message = _copy(moves, **more)
    assert rc == -22 and text in message


@pytest.mark.parametrize("edits,text", [
    ([(0, 4, 0, 0)], "no such sequence"), ([(0, -1, 0, 0)], "no such sequence"), ([(0, 0, 6, 0)], "no such entry"),
    ([(0, 0, 0, 9)], "no such entry"), ([(0, 0, 0, -2)], "no such entry"), ([(1, 0, -1, 0)], "below zero"),
    ([(3, 0, 0, 0)], "no such edit"), ([(0, 0, 1, 1), (0, 0, 1, 2)], "two edits"),
    ([(2, 1, 0, 0), (1, 1, 2, 0)], "two edits"), ([(0, 1, 0, 3), (2, 1, 0, 0)], "two edits"),
    ([(0, 0, 0, 0)] * 129, "more edits")])
def test_pages_edit_refuses(edits, text):
    from mlx_omnia_amd.runtime import library, loader
    flat = ops._int_lines(edits, 4, "edits")
    assert library().omnia_pages_edit(4096, 8192, 4, 6, 9, flat.buffer_info()[0], len(edits), None) == -22
    assert text in loader.last_error()


@pytest.mark.parametrize("change,text", [
    (dict(parent=4), "no such sequence"), (dict(parent=-1), "no such sequence"), (dict(full=7), "outside"),
    (dict(full=6), "no such page"), (dict(rows=17), "outside"), (dict(rows=-1), "outside"), (dict(page=9), "no such page"),
    (dict(page=-1), "no such page"), (dict(kids=[(4, 1)]), "no other sequence"), (dict(kids=[(0, 1)]), "no other sequence"),
    (dict(kids=[(1, 1), (1, 2)]), "named twice"), (dict(kids=[(1, 1), (2, 1)]), "named twice"),
    (dict(kids=[(1, 3)]), "no other page"), (dict(kids=[(1, 9)]), "no other page"), (dict(rows=0), "no other page"),
    (dict(kids=[(1, 1)] * 129), "more children"), (dict(width=0), "bad tables")])
def test_pages_fork_refuses(change, text):
    from mlx_omnia_amd.runtime import library, loader
    case = dict(width=6, parent=0, full=2, page=3, rows=5, kids=[(1, 1)], **{}) | change
    kids = ops._int_lines(case["kids"], 2, "kids")
    assert library().omnia_pages_fork(4096, 8192, 1, 9, 2, 16, 64, 4096, 8192, 4, case["width"], case["parent"],
                                      case["full"], case["page"], case["rows"], kids.buffer_info()[0], len(kids) // 2, None) == -22
    assert text in loader.last_error()


def test_lines_of_numbers():
    assert list(ops._int_lines([], 3, "moves")) == [] and list(ops._int_lines([(1, 2, 3)], 3, "moves")) == [1, 2, 3]
    for bad in ([(1, 2)], [(1, 2, 1 << 31)], [(1, 2, -(1 << 40))], [(1.5, 2, 3)], [1, 2, 3], [(1, 2, 3), (1,)]):
        with pytest.raises(ValueError, match="moves"):
            ops._int_lines(bad, 3, "moves")


def test_another_batch_of_the_same_sequences_keeps_up():
    cache = small()
    a = cache.open(15)
    one, two = cache.batch([a]), cache.batch([a], tokens=2)
    assert cache.ready(one) == 16 and cache.ready(two) == 17 and len(cache.pages_of(a)) == 2
    for _ in range(17):
        cache.ready(one)
        cache.advance(one)
    assert cache.ready(two) == 34 and len(cache.pages_of(a)) == 3


def test_the_steps_arguments_are_laid_out_as_declared():
    import ctypes
    import re
    from pathlib import Path

    from mlx_omnia_amd.runtime.loader import BatchStep

    text = (Path(__file__).resolve().parent.parent / "include" / "omnia_hip.h").read_text()
    body = re.search(r"typedef struct \{([^}]*)\} omnia_attention_batch_step_t;", text).group(1)
    declared = []
    for line in body.replace("const ", "").split(";"):
        kind, _, names = line.strip().partition(" ")
        for name in filter(None, (n.strip() for n in names.split(","))):
            pointer = name.startswith("*")
            declared.append((name.lstrip("*"), ctypes.c_void_p if pointer else
                             {"int64_t": ctypes.c_int64, "float": ctypes.c_float}[kind]))
    assert declared == list(BatchStep._fields_)


def _kept(**change):
    """The host's part of a cache of six pages of 16 rows and five sequences of at most four."""
    state = dict(tables=np.array([[0, 1, 2, -1], [0, 4, -1, -1], *[[-1] * 4] * 3], dtype=np.int32),
                 rows=np.array([37, 20, 0, 0, 0]), held=np.array([3, 2, 0, 0, 0]), refs=np.array([2, 1, 1, 0, 1, 0]),
                 generation=np.zeros(5, dtype=np.int64), open=np.array([1, 1, 0, 0, 0], dtype=np.uint8))
    for name, (at, value) in change.items():
        state[name][at] = value
    return state


def _call_kept(name, state, *args):
    import ctypes

    from mlx_omnia_amd.runtime import library
    from mlx_omnia_amd.runtime.loader import PagedCache
    cache = PagedCache(4096, 8192, 4096, 8192, *(state[n].ctypes.data for n in ("tables", "rows", "held", "refs", "generation", "open")),
                       1, 6, 2, 16, 64, 5, 4)
    return getattr(library(), name)(ctypes.addressof(cache), *args, None)


@pytest.mark.parametrize("change,parent,count,text", [
    ({}, 2, 1, "2 is not open"), ({}, -1, 1, "-1 is not open"), ({}, 5, 1, "5 is not open"), ({}, 0, -1, "no forks"),
    ({}, 0, 4, "4 more sequences are asked for, 3 of 5 are not open"),
    ({}, 0, 3, "3 more pages are needed, 2 of 6 are free"),
    (dict(held=(0, 2)), 0, 1, "more rows than pages"), (dict(held=(0, 5)), 0, 1, "more rows than pages"),
    (dict(tables=((0, 1), -1)), 0, 1, "outside the pool"), (dict(tables=((0, 0), 6)), 0, 1, "outside the pool"),
    (dict(tables=((0, 2), 6)), 0, 1, "no such page")])
def test_paged_cache_fork_refuses(change, parent, count, text):
    """And leaves everything as it was."""
    from mlx_omnia_amd.runtime import loader
    state, before = _kept(**change), _kept(**change)
    kids = np.zeros(2 * max(count, 0), dtype=np.int32)
    assert _call_kept("omnia_paged_cache_fork", state, parent, count, kids.ctypes.data) == -22
    assert text in loader.last_error()
    assert all(np.array_equal(state[n], before[n]) for n in state)


@pytest.mark.parametrize("change,gone,text", [
    ({}, [2], "2 is not open"), ({}, [0, 1, -1], "-1 is not open"), ({}, [1, 5], "5 is not open"),
    ({}, [0, 1, 0], "named twice"), (dict(held=(1, 5)), [0, 1], "more pages than its table")])
def test_paged_cache_free_refuses(change, gone, text):
    """And leaves everything as it was."""
    from mlx_omnia_amd.runtime import loader
    state, before = _kept(**change), _kept(**change)
    assert _call_kept("omnia_paged_cache_free", state, np.array(gone, dtype=np.int32).ctypes.data, len(gone)) == -22
    assert text in loader.last_error()
    assert all(np.array_equal(state[n], before[n]) for n in state)


@pytest.mark.parametrize("change,rows,text", [
    ({}, -1, "fewer than no rows"), ({}, 65, "at most 64 rows, not 65"), ({}, 1 << 62, "at most 64"),
    ({}, 33, "3 more pages are needed, 2 of 6 are free"),
    (dict(open=(slice(None), 1)), 1, "1 more sequences are asked for, 0 of 5 are not open")])
def test_paged_cache_open_refuses(change, rows, text):
    """And leaves everything as it was."""
    from mlx_omnia_amd.runtime import loader
    state, before = _kept(**change), _kept(**change)
    which = np.zeros(1, dtype=np.int32)
    assert _call_kept("omnia_paged_cache_open", state, rows, which.ctypes.data) == -22
    assert text in loader.last_error()
    assert all(np.array_equal(state[n], before[n]) for n in state)


def test_an_empty_sequence_and_a_pool_that_is_packed():
    """What launches nothing."""
    state = _kept()
    which, live = np.zeros(1, dtype=np.int32), np.zeros(1, dtype=np.int64)
    assert _call_kept("omnia_paged_cache_open", state, 0, which.ctypes.data) == 0 and which[0] == 2
    assert state["open"].tolist() == [1, 1, 1, 0, 0] and state["generation"].tolist() == [0, 0, 1, 0, 0]
    state["refs"][:] = [2, 1, 1, 1, 0, 0]
    state["tables"][1, 1] = 3
    before = {n: a.copy() for n, a in state.items()}
    assert _call_kept("omnia_paged_cache_compact", state, live.ctypes.data) == 0 and live[0] == 4
    assert all(np.array_equal(state[n], before[n]) for n in state)


def test_no_forks_and_nothing_freed():
    state = _kept()
    assert _call_kept("omnia_paged_cache_fork", state, 0, 0, None) == 0
    assert _call_kept("omnia_paged_cache_free", state, None, 0) == 0


def test_the_caches_host_part_is_laid_out_as_declared():
    import ctypes
    import re
    from pathlib import Path

    from mlx_omnia_amd.runtime.loader import PagedCache

    text = (Path(__file__).resolve().parent.parent / "include" / "omnia_hip.h").read_text()
    body = re.search(r"typedef struct \{([^}]*)\} omnia_paged_cache_t;", text).group(1)
    declared = []
    for line in body.split(";"):
        kind, _, names = line.strip().partition(" ")
        for name in filter(None, (n.strip() for n in names.split(","))):
            pointer = name.startswith("*") or kind.endswith("*")
            declared.append((name.lstrip("*"), ctypes.c_void_p if pointer else {"int64_t": ctypes.c_int64}[kind]))
    assert declared == list(PagedCache._fields_), declared


def test_tables_in_another_order():
    """Arrays as numpy may lay them out: by columns, of other kinds."""
    pool = torch.zeros((1, 6, 2, 16, 8))
    cache = PagedKVCache(pool, pool.clone(), tables=np.asfortranarray([[0, 1], [2, -1]]), lengths=np.array([20.0, 3.0]), opened=[0, 1])
    assert cache._tables.flags.c_contiguous and cache.rows(0) == 20 and cache.pages_of(0) == [0, 1]
    with pytest.raises(ValueError, match="asked for"):
        cache.fork(0, 1 << 60)


@pytest.mark.parametrize("fails", ["_copy", "_edit"])
@pytest.mark.parametrize("call", ["reserve", "ready", "fork", "truncate"])
def test_a_launch_that_fails_leaves_the_hosts_part_as_it_was(monkeypatch, call, fails):
    cache = small(pages=20)
    parent = cache.open(40)
    kids = cache.fork(parent, 2)
    for s in (parent, *kids):
        cache.truncate(s, 30)   # in a page that the three of them share
    batch = cache.batch([parent, *kids], tokens=20)
    calls = dict(reserve=lambda: cache.reserve(parent, 50), ready=lambda: cache.ready(batch),
                 fork=lambda: cache.fork(parent, 2, share=False), truncate=lambda: cache.truncate(parent, 9))
    names = "_tables", "_rows", "_held", "_refs", "_generation", "_open"
    before = {name: getattr(cache, name).copy() for name in names}
    if call != "truncate" or fails != "_copy":   # which copies nothing
        def fail(*args, **kwargs):
            raise RuntimeError("not launched")

        with monkeypatch.context() as patch:
            patch.setattr(cache, fails, fail)
            with pytest.raises(RuntimeError, match="not launched"):
                calls[call]()
        for name in names:
            assert np.array_equal(getattr(cache, name), before[name]), name
    calls[call]()
    assert any(not np.array_equal(getattr(cache, name), before[name]) for name in names)
    for s in np.flatnonzero(cache._open):
        assert cache.tables[s].tolist() == cache._tables[s].tolist() and cache.lengths[s] == cache.rows(s)


# Where the kernels read ------------------------------------------------------------------------


@pytest.fixture
def launches(monkeypatch):
    """A device's path on CPU tensors: what the library would be called with, and nothing run."""
    import types

    from mlx_omnia_amd.kernels.attention import batch, pages
    from mlx_omnia_amd.runtime.loader import BatchStep, PagedCache

    seen = []

    def call(name, *args):
        kind = {"omnia_attention_batch_step": BatchStep, "omnia_paged_cache_fork": PagedCache,
                "omnia_paged_cache_open": PagedCache, "omnia_paged_cache_free": PagedCache,
                "omnia_paged_cache_compact": PagedCache}.get(name)
        seen.append((name, kind.from_buffer_copy(kind.from_address(args[0])) if kind else args))

    for module in (batch, pages):
        monkeypatch.setattr(module, "hip_device", lambda *tensors: True)
    monkeypatch.setattr(ops, "on_rocm", lambda *tensors: True)
    monkeypatch.setattr(ops, "_stream_here", lambda index: 0)
    monkeypatch.setattr(ops, "library", lambda: types.SimpleNamespace(omnia_attention_batch_step_bytes=lambda *a: 256))
    monkeypatch.setattr(ops, "call", call)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return seen


def _taken_up(layers=2):
    shape = (layers, 8, 2, 16, 64)
    return PagedKVCache(torch.zeros(shape, dtype=torch.bfloat16), torch.zeros(shape, dtype=torch.bfloat16),
                        tables=np.array([[0, 1, -1], [0, 2, -1], [-1, -1, -1]]), lengths=np.array([20, 21, 0]), opened=[0, 1])


def _declared(cache):
    gen = torch.Generator().manual_seed(1)
    made = lambda *shape, dtype=torch.bfloat16: torch.randn(shape, generator=gen).to(dtype)  # noqa: E731
    parts = dict(query_weight=made(64), key_weight=made(64), sinks=made(8), cos_rows=made(48, 32, dtype=torch.float32),
                 sin_rows=made(48, 32, dtype=torch.float32))
    step = BatchAttentionStep(cache, layer=1, heads=8, kv_heads=2, head_dim=64, scale=0.1, dtype=torch.bfloat16,
                              query_weight=parts["query_weight"], key_weight=parts["key_weight"], rotary_pairs=32,
                              angles=AngleTable(parts["cos_rows"], parts["sin_rows"]), sinks=parts["sinks"])
    parts |= dict(keys=cache.keys, values=cache.values, tables=cache.tables, lengths=cache.lengths)
    return step, parts, [made(2, n * 64) for n in (8, 2, 2)]


@pytest.mark.parametrize("name", ["query_weight", "key_weight", "sinks", "cos_rows", "sin_rows", "keys", "values", "tables",
                                  "lengths"])
def test_a_step_reads_its_tensors_where_they_lie_by_now(launches, name):
    """A module that is moved, or its parameters sharded, gives the same tensors other memory."""
    cache = _taken_up()
    step, parts, raw = _declared(cache)
    batch = cache.batch([0, 1])
    for call in (step, step.project):
        for _ in range(2):
            call(batch, *raw)
            parts[name].data = parts[name].data.clone()
            call(batch, *raw)
            got, layer = launches[-1][1], cache.keys[0].numel() * 2
            for field, t in parts.items():
                assert getattr(got, field) == t.data_ptr() + (layer if field in ("keys", "values") else 0), field


def test_a_steps_tensors_are_checked_where_they_lie_by_now(launches):
    cache = _taken_up()
    step, parts, raw = _declared(cache)
    batch = cache.batch([0, 1])
    for name in ("query_weight", "key_weight", "sinks", "cos_rows"):
        held = parts[name].data
        others = [held.double(), held[..., :4].clone()]
        if name.endswith("weight"):
            others.append(held.repeat(2)[1:65])   # off the 16 bytes that are read at a time
        for other in others:
            step(batch, *raw)
            count = len(launches)
            parts[name].data = other
            with pytest.raises(ValueError):
                step(batch, *raw)
            assert len(launches) == count
            parts[name].data = held
    parts["query_weight"].data = torch.empty(0, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        step(batch, *raw)
    emptied = parts["key_weight"]
    parts["query_weight"].data = emptied.data.clone()
    step(batch, *raw)
    emptied.untyped_storage().resize_(0)   # as a sharded parameter's between its uses: no address
    with pytest.raises(ValueError):
        step(batch, *raw)


@pytest.mark.parametrize("scale,served", [(0.1, True), (2.0 ** -126, True), (1e-39, False), (1e-50, False), (0.0, False),
                                          (-1.0, False), (1e38, True), (3e38, False), (1e39, False), (float("nan"), False)])
def test_scales_that_32_bits_do_not_hold(launches, scale, served):
    """They go to the Core chain, and not to kernels that refuse every call."""
    step = BatchAttentionStep(_taken_up(), layer=0, heads=8, kv_heads=2, head_dim=64, scale=scale, dtype=torch.bfloat16)
    assert (type(step.strategy) is not DefaultBatchAttentionStep) == served


@pytest.mark.parametrize("scale,rc", [(0.1, 0), (1e38, 0), (3e38, -22), (1e39, -22), (0.0, -22), (-1.0, -22), (float("nan"), -22)])
def test_attention_batch_refuses_scales(scale, rc):
    from mlx_omnia_amd.runtime import library
    at = 4096   # of no tokens: nothing is looked at
    assert library().omnia_attention_batch(at, 0, at, at, 8, 16, at, 2, 4, at, at, 0, at, 0, 0, 0, 0, 0, 8, 2, 64, None, scale,
                                           None, 0, at, None) == rc


def test_sinks_that_do_not_lie_together_are_read_as_they_are_now(launches):
    import ctypes

    cache = _taken_up()
    table = torch.arange(24, dtype=torch.float32).bfloat16().reshape(8, 3)
    step = BatchAttentionStep(cache, layer=0, heads=8, kv_heads=2, head_dim=64, scale=0.1, dtype=torch.bfloat16,
                              sinks=table[:, 1])
    assert type(step.strategy).__name__ == "HipBatchAttentionStep"
    batch = cache.batch([0, 1])
    raw = [torch.zeros(2, n * 64, dtype=torch.bfloat16) for n in (8, 2, 2)]
    read = []

    def call(name, address, stream):
        from mlx_omnia_amd.runtime.loader import BatchStep
        read.append(list((ctypes.c_uint16 * 8).from_address(BatchStep.from_address(address).sinks)))

    with pytest.MonkeyPatch.context() as patch:
        patch.setattr(ops, "call", call)
        for change in (0.0, 1.0, 7.0):
            table += change
            step(batch, *raw)
            assert read[-1] == table[:, 1].contiguous().view(torch.uint16).tolist()


def test_a_plan_of_no_tokens(launches):
    cache = _taken_up()
    none = torch.empty((0, 2), dtype=torch.int32)
    plan = ops.BatchStepPlan(None, None, None, cache.keys[0], cache.values[0], cache.tables, cache.lengths, none,
                             torch.empty((0, 4), dtype=torch.int32), heads=8, prefix=0, prefix_sequence=0, scale=0.1, eps=1e-6)
    assert plan(*(torch.empty((0, n * 64), dtype=torch.bfloat16) for n in (8, 2, 2)), 1).shape == (0, 8, 64)
    assert launches[-1][1].tokens == 0


def test_a_caches_calls_name_its_pool_where_it_lies_by_now(launches):
    cache = _taken_up()
    calls = [lambda: cache.fork(0), lambda: cache.open(3), lambda: cache.free(1), cache.compact]
    for name in ("keys", "values", "tables", "lengths"):
        held = getattr(cache, name)
        held.data = held.data.clone()
        for call in calls if name == "tables" else calls[:2]:
            call()
            got = launches[-1][1]
            assert all(getattr(got, n) == getattr(cache, n).data_ptr() for n in ("keys", "values", "tables", "lengths"))
    cache.values = cache.values.clone()
    cache.fork(0)
    assert launches[-1][1].values == cache.values.data_ptr()
    cache.reserve(0, 40)   # pages in the torch order of things, edited by the library
    assert launches[-1][0] == "omnia_pages_edit" and launches[-1][1][0] == cache.tables.data_ptr()
    held, count = cache.keys.data, len(launches)
    for other in (held.view(torch.float16), held[:1].clone(), held[:, :4].clone()):
        cache.keys.data = other
        for call in calls:
            with pytest.raises(ValueError):
                call()
    assert len(launches) == count
    cache.keys.data = held
    cache.fork(0)
