"""A cache of pages that many sequences share, and the attention of a batch over it.

What a program does that answers one prompt many times: it forks a sequence, frees and
compacts what it no longer needs, writes a batch's new keys and values into the pages, and
takes a layer's attention for all of them, the rows that they share once for all.

`own` says which side `run` takes: the plain one, in elementary torch operations, or the
framework's calls. Both work on the same pool, tables and lengths, so a case's outputs are
the tables, the pages and the contexts that either leaves.

The lengths of a case's sequences follow from its sizes alone (`_before`, `_tokens`); the
pages they lie on, and every value, from the seed.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DEVICE = "cuda"
EPS = 1e-6
BASE = 1e6


def listed() -> list[dict]:
    return [
        # One answer forked off a short prompt, in a small model: a few pages' ends, all latency.
        dict(name="fork_one", kind="fork", layers=4, kv_heads=2, head_dim=64, page_rows=16, rows=37, count=1),
        # Sixteen answers sampled from one prompt, all layers of a cache (36).
        dict(name="fork_samples", kind="fork", layers=36, kv_heads=8, head_dim=128, page_rows=64, rows=8033,
             count=16),
        # A batch turns over: half of the sequences end, the pool is packed, others begin; twice.
        dict(name="compact_turnover", kind="compact", layers=16, kv_heads=8, head_dim=128, page_rows=64,
             sequences=12, rows=1200),
        # A decode step's rows into the pages: 64 sequences of one token.
        dict(name="write_decode", kind="write", batch=64, heads=32, kv_heads=8, head_dim=128, pairs=64, norms=True,
             page_rows=64, prefix=2048, own=300, tokens=1),
        # Prompts of different lengths into the pages, no norms, half a head rotated.
        dict(name="write_prompts", kind="write", batch=7, heads=64, kv_heads=8, head_dim=64, pairs=16, norms=False,
             page_rows=16, prefix=0, own=90, tokens=1100),
        # The smallest step: two answers, little behind them.
        dict(name="step_pair", kind="step", batch=2, heads=8, kv_heads=2, head_dim=128, pairs=64, norms=True,
             sinks=False, page_rows=16, prefix=208, own=21, tokens=1),
        # Sixteen answers sampled from a prompt of 8,192 rows.
        dict(name="step_samples", kind="step", batch=16, heads=32, kv_heads=8, head_dim=128, pairs=64, norms=True,
             sinks=False, page_rows=64, prefix=8192, own=700, tokens=1),
        # Many requests behind one system prompt, groups of eight.
        dict(name="step_system_prompt", kind="step", batch=96, heads=32, kv_heads=4, head_dim=128, pairs=64,
             norms=True, sinks=False, page_rows=32, prefix=4000, own=500, tokens=1),
        # A long document asked about by 128 requests: the largest.
        dict(name="step_document", kind="step", batch=128, heads=32, kv_heads=8, head_dim=128, pairs=64, norms=True,
             sinks=False, page_rows=64, prefix=32768, own=1024, tokens=1),
        # A layer with sinks, 64 heads of 64, an odd batch, small pages.
        dict(name="step_sinks", kind="step", batch=33, heads=64, kv_heads=8, head_dim=64, pairs=32, norms=False,
             sinks=True, page_rows=16, prefix=2000, own=333, tokens=1),
        # Requests that share nothing, of very different lengths.
        dict(name="step_unshared", kind="step", batch=24, heads=32, kv_heads=8, head_dim=128, pairs=64, norms=True,
             sinks=False, page_rows=32, prefix=0, own=16000, tokens=1),
        # Several questions of different lengths, taken in at once behind one document.
        dict(name="step_questions", kind="step", batch=9, heads=32, kv_heads=8, head_dim=128, pairs=64, norms=True,
             sinks=False, page_rows=64, prefix=4096, own=60, tokens=400),
    ]


def _log(rng, low: int, high: int) -> int:
    """A whole number in [low, high], spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(["fork", "compact", "write", "step", "step", "step", "prompts"])
    page_rows = rng.choice([16, 32, 64, 64, 128, 256])
    kv_heads, head_dim = rng.choice([1, 2, 4, 8, 8]), rng.choice([64, 128, 128])
    if kind == "fork":
        return dict(kind=kind, layers=_log(rng, 1, 36), kv_heads=kv_heads, head_dim=head_dim, page_rows=page_rows,
                    rows=_log(rng, 1, 8000), count=_log(rng, 1, 16))
    if kind == "compact":
        return dict(kind=kind, layers=_log(rng, 1, 16), kv_heads=kv_heads, head_dim=head_dim, page_rows=page_rows,
                    sequences=2 * rng.randint(1, 6), rows=_log(rng, 1, 1200))
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8, 8])
    shape = dict(heads=heads, kv_heads=kv_heads, head_dim=head_dim, pairs=rng.choice([head_dim // 2, head_dim // 4]),
                 norms=rng.random() < 0.6, page_rows=page_rows)
    if kind == "write":
        prompts = rng.random() < 0.5
        return dict(kind=kind, batch=_log(rng, 1, 8 if prompts else 128), prefix=page_rows * rng.randint(0, 8),
                    own=_log(rng, 1, 300), tokens=_log(rng, 2, 1100) if prompts else 1, **shape)
    shape["sinks"] = rng.random() < 0.3
    if kind == "prompts":
        return dict(kind="step", batch=_log(rng, 1, 9), prefix=page_rows * rng.randint(0, 4096 // page_rows),
                    own=_log(rng, 1, 500), tokens=_log(rng, 2, 400), **shape)
    if rng.random() < 0.2:
        return dict(kind="step", batch=_log(rng, 1, 24), prefix=0, own=_log(rng, 1, 16000), tokens=1, **shape)
    return dict(kind="step", batch=_log(rng, 1, 128), prefix=page_rows * _log(rng, 1, 32768 // page_rows),
                own=_log(rng, 1, 1024), tokens=1, **shape)


# Sizes that follow from a case ------------------------------------------------------------


def _spread(count: int, high: int, step: int) -> list[int]:
    """`count` different-looking numbers in [1, high], the highest among them."""
    return [high - (i * step * 131) % high for i in range(count)]


def _before(case: dict) -> list[int]:
    """Rows that each sequence holds before the step."""
    return [case["prefix"] + n - 1 for n in _spread(case["batch"], case["own"], 61)]


def _tokens(case: dict) -> list[int]:
    """New tokens of each sequence."""
    return [1] * case["batch"] if case["tokens"] == 1 else _spread(case["batch"], case["tokens"], 17)


def _turnover_rows(case: dict) -> list[int]:
    half = _spread(case["sequences"] // 2, case["rows"], 29)
    return half + half


def _pages_for(rows: int, page_rows: int) -> int:
    return -(-rows // page_rows)


# Inputs -----------------------------------------------------------------------------------


def _pool(gen, layers: int, pages: int, case: dict) -> torch.Tensor:
    pool = torch.empty((layers, pages, case["kv_heads"], case["page_rows"], case["head_dim"]), dtype=BF16,
                       device=DEVICE)
    for layer in pool:
        layer.copy_(torch.randn(layer.shape, generator=gen, device=DEVICE, dtype=F32))
    return pool


def _inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    order = random.Random(seed)
    size, kind = case["page_rows"], case["kind"]
    if kind == "fork":
        held, layers = _pages_for(case["rows"], size), case["layers"]
        pages, sequences, width = held + case["count"] + 3, 2 + case["count"], held + 1
        ids = order.sample(range(pages), held + 1)
        tables = np.full((sequences, width), -1, dtype=np.int32)
        tables[0, :held], tables[1, 0] = ids[:held], ids[held]
        lengths = np.zeros(sequences, dtype=np.int32)
        lengths[:2] = case["rows"], 1
        opened = [0, 1]
    elif kind == "compact":
        rows, layers = _turnover_rows(case), case["layers"]
        held = [_pages_for(n, size) for n in rows]
        pages, sequences, width = sum(held) + 2, len(rows), max(held) + 1
        tables = np.full((sequences, width), -1, dtype=np.int32)
        first = 0
        for i, n in enumerate(held):
            tables[i, :n] = np.arange(first, first + n)
            first += n
        lengths = np.asarray(rows, dtype=np.int32)
        opened = list(range(sequences))
    else:
        before, tokens, layers = _before(case), _tokens(case), 1
        shared = case["prefix"] // size
        held = [_pages_for(b + t, size) for b, t in zip(before, tokens)]
        pages, sequences, width = shared + sum(n - shared for n in held) + 3, case["batch"] + 1, max(held) + 1
        ids = order.sample(range(pages), pages)
        tables = np.full((sequences, width), -1, dtype=np.int32)
        at = shared
        for i, n in enumerate(held):
            tables[i, :shared] = ids[:shared]
            tables[i, shared:n] = ids[at : at + n - shared]
            at += n - shared
        lengths = np.zeros(sequences, dtype=np.int32)
        lengths[: case["batch"]] = before
        opened = list(range(case["batch"]))
    inputs = dict(tables=tables, lengths=lengths, opened=opened, keys=_pool(gen, layers, pages, case),
                  values=_pool(gen, layers, pages, case))
    if kind in ("fork", "compact"):
        return inputs
    normal = lambda *shape: torch.randn(shape, generator=gen, device=DEVICE)  # noqa: E731
    d, total = case["head_dim"], sum(tokens)
    inputs["q"] = normal(total, case["heads"] * d).to(BF16)
    inputs["k"] = normal(total, case["kv_heads"] * d).to(BF16)
    inputs["v"] = normal(total, case["kv_heads"] * d).to(BF16)
    gains = [(1 + 0.1 * normal(d)).to(BF16) for _ in range(2)]
    inputs["qw"], inputs["kw"] = gains if case["norms"] else (None, None)
    theta = (torch.arange(max(b + t for b, t in zip(before, tokens)), dtype=F64, device=DEVICE)[:, None]
             * torch.exp(-math.log(BASE) * torch.arange(case["pairs"], dtype=F64, device=DEVICE) / case["pairs"]))
    inputs["cos"], inputs["sin"] = torch.cos(theta).to(F32), torch.sin(theta).to(F32)
    inputs["sinks"] = normal(case["heads"]).to(BF16) if case.get("sinks") else None
    return inputs


def prepare(case: dict, seed: int) -> dict:
    state = dict(_inputs(case, seed), case=case, own=own, kids=[])
    if not own:
        refs = np.zeros(state["keys"].shape[1], dtype=np.int64)
        np.add.at(refs, state["tables"][state["tables"] >= 0], 1)
        state.update(refs=refs, device_tables=torch.from_numpy(state["tables"].copy()).to(DEVICE),
                     device_lengths=torch.from_numpy(state["lengths"].copy()).to(DEVICE))
        if case["kind"] in ("write", "step"):
            state.update(_plain_positions(state))
        return state
    import __graft_entry__

    __graft_entry__.load_package()
    from mlx_omnia_amd.kernels.attention import BatchAttentionStep, PagedKVCache
    from mlx_omnia_amd.kernels.qkv_rope import AngleTable

    cache = PagedKVCache(state["keys"], state["values"], tables=state["tables"], lengths=state["lengths"],
                         opened=state["opened"])
    state["cache"] = cache
    if case["kind"] in ("write", "step"):
        state["batch"] = cache.batch(state["opened"], tokens=_tokens(case))
        state["step"] = BatchAttentionStep(
            cache, layer=0, heads=case["heads"], kv_heads=case["kv_heads"], head_dim=case["head_dim"],
            scale=case["head_dim"] ** -0.5, dtype=BF16, query_weight=state["qw"], key_weight=state["kw"], eps=EPS,
            rotary_pairs=case["pairs"], angles=AngleTable(state["cos"], state["sin"]), sinks=state["sinks"])
    return state


def run(state: dict):
    kind = state["case"]["kind"]
    if not state["own"]:
        return {"fork": _plain_fork, "compact": _plain_compact, "write": _plain_write, "step": _plain_step}[kind](state)
    cache = state["cache"]
    if kind == "fork":
        # The answers of the pass before end, and as many new ones begin.
        if state["kids"]:
            cache.free(state["kids"])
        state["kids"] = cache.fork(0, state["case"]["count"])
        return cache.tables, cache.lengths, cache.keys, cache.values
    if kind == "compact":
        rows = _turnover_rows(state["case"])
        half = len(rows) // 2
        for group in (range(half), range(half, 2 * half)):
            cache.free(list(group))
            cache.compact()
            for sequence in group:
                cache.open(rows[sequence])
        return cache.tables, cache.lengths, cache.keys, cache.values
    if kind == "write":
        queries = state["step"].project(state["batch"], state["q"], state["k"], state["v"])
        return queries, cache.keys, cache.values
    context = state["step"](state["batch"], state["q"], state["k"], state["v"])
    return context, cache.keys, cache.values


# The plain form ---------------------------------------------------------------------------


def _lowest_free(state: dict, count: int) -> np.ndarray:
    return np.flatnonzero(state["refs"] == 0)[:count]


def _plain_free(state: dict, sequences: list[int]) -> None:
    for s in sequences:
        row = state["tables"][s]
        np.subtract.at(state["refs"], row[row >= 0], 1)
    state["tables"][sequences] = -1
    state["lengths"][sequences] = 0
    state["device_tables"][sequences] = -1
    state["device_lengths"][sequences] = 0


def _plain_fork(state: dict):
    case, tables, size = state["case"], state["tables"], state["case"]["page_rows"]
    if state["kids"]:
        _plain_free(state, state["kids"])
    kids = list(range(2, 2 + case["count"]))
    full, rest = divmod(int(state["lengths"][0]), size)
    tables[kids, :full] = tables[0, :full]
    if rest:
        fresh = _lowest_free(state, len(kids))
        tables[kids, full] = fresh
        to, page = torch.from_numpy(fresh).to(DEVICE), int(tables[0, full])
        for pool in (state["keys"], state["values"]):
            pool[:, to, :, :rest] = pool[:, page, :, :rest].unsqueeze(1)
    for s in kids:
        np.add.at(state["refs"], tables[s][tables[s] >= 0], 1)
    state["lengths"][kids] = state["lengths"][0]
    state["device_tables"][kids] = torch.from_numpy(tables[kids]).to(DEVICE)
    state["device_lengths"][kids] = int(state["lengths"][0])
    state["kids"] = kids
    return state["device_tables"], state["device_lengths"], state["keys"], state["values"]


def _plain_compact(state: dict):
    rows, size = _turnover_rows(state["case"]), state["case"]["page_rows"]
    half, tables, refs = len(rows) // 2, state["tables"], state["refs"]
    for group in (range(half), range(half, 2 * half)):
        _plain_free(state, list(group))
        live = int((refs > 0).sum())
        source = np.flatnonzero(refs > 0)
        source, target = source[source >= live], np.flatnonzero(refs[:live] == 0)
        if len(source):
            at, to = torch.from_numpy(source).to(DEVICE), torch.from_numpy(target).to(DEVICE)
            for pool in (state["keys"], state["values"]):
                pool[:, to] = pool[:, at]
            names = np.arange(len(refs) + 1, dtype=np.int32)   # the last for -1
            names[-1], names[source] = -1, target
            tables[:] = names[tables]
            state["device_tables"].copy_(torch.from_numpy(names).to(DEVICE)[state["device_tables"].long()])
            refs[target], refs[source] = refs[source], 0
        for s in group:
            fresh = _lowest_free(state, _pages_for(rows[s], size))
            refs[fresh] = 1
            tables[s, : len(fresh)] = fresh
            state["lengths"][s] = rows[s]
            state["device_tables"][s] = torch.from_numpy(tables[s]).to(DEVICE)
            state["device_lengths"][s] = rows[s]
    return state["device_tables"], state["device_lengths"], state["keys"], state["values"]


def _plain_positions(state: dict) -> dict:
    """Each token's position, page and row in it, on the device."""
    case = state["case"]
    positions, pages = [], []
    for i, (b, t) in enumerate(zip(_before(case), _tokens(case))):
        at = np.arange(b, b + t)
        positions.append(at)
        pages.append(state["tables"][i, at // case["page_rows"]])
    at = torch.from_numpy(np.concatenate(positions)).to(DEVICE)
    return dict(positions=at, page_of=torch.from_numpy(np.concatenate(pages)).long().to(DEVICE),
                row_of=at % case["page_rows"])


def _project(state: dict, kind):
    """(queries, keys, values) [N, heads, D] of the new tokens in `kind`, before any rounding."""
    case, d = state["case"], state["case"]["head_dim"]
    p = case["pairs"]
    cos = state["cos"][state["positions"]].to(kind)[:, None]
    sin = state["sin"][state["positions"]].to(kind)[:, None]
    parts = []
    for name, gain in (("q", "qw"), ("k", "kw")):
        x = state[name].to(kind).unflatten(-1, (-1, d))
        if state[gain] is not None:
            x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * state[gain].to(kind)
        a, b = x[..., :p], x[..., p : 2 * p]
        parts.append(torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * p :]], dim=-1))
    return *parts, state["v"].to(kind).unflatten(-1, (-1, d))


def _plain_write(state: dict):
    q, k, v = _project(state, F32)
    state["keys"][0, state["page_of"], :, state["row_of"]] = k.to(BF16)
    state["values"][0, state["page_of"], :, state["row_of"]] = v.to(BF16)
    return q.to(BF16), state["keys"], state["values"]


def _plain_step(state: dict):
    case = state["case"]
    q, k, v = _project(state, F32)
    state["keys"][0, state["page_of"], :, state["row_of"]] = k.to(BF16)
    state["values"][0, state["page_of"], :, state["row_of"]] = v.to(BF16)
    kv, d, size = case["kv_heads"], case["head_dim"], case["page_rows"]
    group, outs, first = case["heads"] // kv, [], 0
    for i, (b, t) in enumerate(zip(_before(case), _tokens(case))):
        rows = b + t
        pages = state["device_tables"][i, : _pages_for(rows, size)].long()
        keys, values = (pool[0, pages].transpose(0, 1).reshape(kv, -1, d)[:, :rows].to(F32)
                        for pool in (state["keys"], state["values"]))
        mine = q[first : first + t].unflatten(1, (kv, group)).permute(1, 2, 0, 3).reshape(kv, group * t, d)
        scores = torch.matmul(mine, keys.transpose(1, 2).contiguous()).unflatten(1, (group, t)) * d ** -0.5
        if t > 1:
            seen = torch.arange(rows, device=DEVICE)[None] <= torch.arange(b, rows, device=DEVICE)[:, None]
            scores = torch.where(seen, scores, torch.full((), -math.inf, device=DEVICE))
        top = scores.amax(dim=-1, keepdim=True)
        if state["sinks"] is not None:
            sink = state["sinks"].to(F32).reshape(kv, group, 1, 1)
            top = torch.maximum(top, sink)
        weights = torch.exp(scores - top)
        total = weights.sum(dim=-1, keepdim=True)
        if state["sinks"] is not None:
            total = total + torch.exp(sink - top)
        context = torch.matmul(weights.flatten(1, 2), values).unflatten(1, (group, t)) / total
        outs.append(context.permute(2, 0, 1, 3).reshape(t, kv * group, d))
        first += t
    return torch.cat(outs).to(BF16), state["keys"], state["values"]


# What a pass cannot do without ------------------------------------------------------------


def work(case: dict) -> dict:
    row = 4 * case["kv_heads"] * case["head_dim"]   # bytes of a key and a value row
    size = case["page_rows"]
    if case["kind"] == "fork":
        rest, table = case["rows"] % size, 4 * _pages_for(case["rows"], size)
        return dict(bytes=case["layers"] * row * rest * (1 + case["count"]) + table * (1 + case["count"]), flops=0)
    if case["kind"] == "compact":
        moved = sum(_pages_for(n, size) for n in _turnover_rows(case))
        return dict(bytes=2 * case["layers"] * row * size * moved, flops=0)
    before, tokens = _before(case), _tokens(case)
    n, d, heads, kv = sum(tokens), case["head_dim"], case["heads"], case["kv_heads"]
    turned = n * (heads + kv) * d
    if case["kind"] == "write":
        return dict(bytes=4 * n * (heads + 2 * kv) * d + 8 * n * case["pairs"], flops=8 * turned)
    attended = sum(b * t + t * (t + 1) // 2 for b, t in zip(before, tokens))
    rows = case["prefix"] + sum(b + t - case["prefix"] for b, t in zip(before, tokens))
    return dict(bytes=row * rows + 2 * n * (2 * heads + 2 * kv) * d + 8 * n * case["pairs"],
                flops=4 * heads * d * attended + 8 * turned)


# The same in 64 bits ----------------------------------------------------------------------


def exact(case: dict, seed: int):
    if case["kind"] in ("fork", "compact"):
        return None   # ids and copies: nothing is computed
    inputs = _inputs(case, seed)
    d, kv, size, pairs = case["head_dim"], case["kv_heads"], case["page_rows"], case["pairs"]
    group = case["heads"] // kv
    keys, values = inputs["keys"].to(F64), inputs["values"].to(F64)
    queries, contexts, first = [], [], 0

    def turned(raw, gain, at):
        x = raw.to(F64).reshape(raw.shape[0], -1, d)
        if gain is not None:
            x = x / torch.sqrt(x.square().sum(dim=-1, keepdim=True) / d + EPS) * gain.to(F64)
        angle = torch.complex(inputs["cos"][at].to(F64), inputs["sin"][at].to(F64))[:, None]
        spun = torch.complex(x[..., :pairs].contiguous(), x[..., pairs : 2 * pairs].contiguous()) * angle
        return torch.cat([spun.real, spun.imag, x[..., 2 * pairs :]], dim=-1)

    for i, (before, count) in enumerate(zip(_before(case), _tokens(case))):
        new = slice(first, first + count)
        at = torch.arange(before, before + count, device=DEVICE)
        table = torch.from_numpy(inputs["tables"][i]).long().to(DEVICE)
        page, row = table[at // size], at % size
        q = turned(inputs["q"][new], inputs["qw"], at)
        keys[0, page, :, row] = turned(inputs["k"][new], inputs["kw"], at)
        values[0, page, :, row] = inputs["v"][new].to(F64).reshape(count, kv, d)
        queries.append(q)
        first += count
        if case["kind"] == "write":
            continue
        rows = before + count
        seen = table[: _pages_for(rows, size)]
        limit = at + 1
        parts = []
        for h in range(kv):
            k = keys[0, seen, h].reshape(-1, d)[:rows]
            v = values[0, seen, h].reshape(-1, d)[:rows]
            for g in range(group):
                head = h * group + g
                s = torch.mv(k, q[0, head])[None] if count == 1 else torch.mm(q[:, head].contiguous(), k.t().contiguous())
                s = s / math.sqrt(d)
                s = s.masked_fill(torch.arange(rows, device=DEVICE)[None] >= limit[:, None], -math.inf)
                if inputs["sinks"] is not None:
                    s = torch.cat([s, inputs["sinks"][head].to(F64).expand(count, 1)], dim=1)
                weight = torch.softmax(s, dim=1)[:, :rows]
                parts.append(torch.mm(weight, v))
        contexts.append(torch.stack(parts, dim=1))
    return (torch.cat(queries) if case["kind"] == "write" else torch.cat(contexts)), keys, values
