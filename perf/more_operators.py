"""Linear attention with a decay for each head, and the norms that stand behind it.

What a layer does whose mixer keeps a state in place of a cache of rows: the mixer itself,
over prompts of many lengths and over steps of one token, the norm and gate of what it
gives, and the join with the residual stream that the next block's norm reads.

    S_t = exp(g_t) S_{t-1} + w_t k_t v_t^T,   o_t = scale * q_t S_t        (mixer)
    y = norm(x) * weight * act(z)  or  norm(x * act(z)) * weight           (gated norm)
    s = a r + b act(gate) norm(x; post),   n = norm(s; pre)                (block norm)

`own` says which side `run` takes: the plain one, in elementary torch operations, or the
framework's calls. A mixer's outputs are the context and the states that it leaves.
"""

from __future__ import annotations

import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DEVICE = "cuda"
EPS = 1e-6
CHUNK = 128   # tokens that the plain mixer takes together


def listed() -> list[dict]:
    return [
        # One request of a small model answers: a token, eight heads of 64. All latency.
        dict(name="step_one", kind="mix", batch=1, tokens=1, heads=8, key_heads=8, key_dim=64, value_dim=64,
             decay="token", strengths=False, fused=True),
        # A decode step of 64 requests, two value heads to a key head.
        dict(name="step_batch", kind="mix", batch=64, tokens=1, heads=32, key_heads=16, key_dim=128, value_dim=128,
             decay="token", strengths=False, fused=True),
        # A decode step of 200 requests in a state-space layer: one key head in eight groups, strengths.
        dict(name="step_states", kind="mix", batch=200, tokens=1, heads=64, key_heads=8, key_dim=128, value_dim=64,
             decay="token", strengths=True, fused=True),
        # A short question to one model: less than a chunk.
        dict(name="prompt_short", kind="mix", batch=1, tokens=37, heads=16, key_heads=16, key_dim=128, value_dim=128,
             decay="token", strengths=False, fused=True),
        # Requests of all lengths taken in at once, single tokens among them.
        dict(name="prompt_ragged", kind="mix", batch=12, tokens=1501, heads=32, key_heads=16, key_dim=128,
             value_dim=128, decay="token", strengths=False, fused=True),
        # Four prompts of a layer whose heads forget at fixed rates.
        dict(name="prompt_fixed", kind="mix", batch=4, tokens=4096, heads=32, key_heads=32, key_dim=128,
             value_dim=128, decay="head", strengths=False, fused=False),
        # A state-space layer's prompt: one key head for all, heads of 64, strengths.
        dict(name="prompt_states", kind="mix", batch=1, tokens=8192, heads=64, key_heads=1, key_dim=128,
             value_dim=64, decay="token", strengths=True, fused=True),
        # A long document, one sequence: the largest.
        dict(name="prompt_long", kind="mix", batch=1, tokens=32768, heads=32, key_heads=32, key_dim=128,
             value_dim=128, decay="token", strengths=False, fused=False),
        # The mixer's output of a decode step of 32 requests.
        dict(name="gated_decode", kind="gated", rows=32, width=4096, group=128, act="silu", gate_first=False),
        # The same of a prompt, a state-space layer's order: gated, then normed in wide groups.
        dict(name="gated_prompt", kind="gated", rows=8192, width=4096, group=512, act="silu", gate_first=True),
        # Two blocks of a decode step of one token meet.
        dict(name="block_decode", kind="block", rows=1, hidden=2560, post=True, gate="none", residual_scale=1.0,
             block_scale=0.7),
        # And of a prompt, the block's output gated token by token.
        dict(name="block_prompt", kind="block", rows=8192, hidden=5120, post=True, gate="rows", residual_scale=0.9,
             block_scale=1.3),
    ]


def _log(rng, low: int, high: int) -> int:
    """A whole number in [low, high], spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(["step", "step", "prompt", "prompt", "prompt", "gated", "block"])
    if kind == "gated":
        group = rng.choice([64, 128, 128, 256, 8 * rng.randint(1, 256)])
        groups = _log(rng, 1, max(1, 8192 // group))
        return dict(kind="gated", rows=_log(rng, 1, 8192), width=group * groups, group=group,
                    act=rng.choice(["silu", "sigmoid"]), gate_first=rng.random() < 0.4)
    if kind == "block":
        return dict(kind="block", rows=_log(rng, 1, 8192), hidden=8 * _log(rng, 8, 640), post=rng.random() < 0.7,
                    gate=rng.choice(["none", "none", "hidden", "rows"]), residual_scale=rng.choice([1.0, 0.9, 3.5]),
                    block_scale=rng.choice([1.0, 0.5, 1.3]))
    key_heads = _log(rng, 1, 32)
    heads = key_heads * rng.choice([n for n in (1, 1, 2, 4, 8, 64) if n * key_heads <= 64])
    case = dict(kind="mix", heads=heads, key_heads=key_heads, key_dim=rng.choice([64, 128, 128]),
                value_dim=rng.choice([64, 128, 128]), decay=rng.choice(["token", "token", "head"]),
                strengths=rng.random() < 0.4, fused=rng.random() < 0.5)
    if kind == "step":
        return dict(case, batch=_log(rng, 1, min(256, 8192 // heads)), tokens=1)
    batch = _log(rng, 1, 16)
    return dict(case, batch=batch, tokens=_log(rng, 2, min(32768, 32768 * 32 // (heads * batch))))


def _lengths(case: dict) -> list[int]:
    """New tokens of each sequence: as many, or different ones down to one token."""
    batch, high = case["batch"], case["tokens"]
    if high == 1 or case["decay"] == "head":
        return [high] * batch
    return [high if i == 0 else 1 if i == 1 else 1 + (high - 1 - i * 131 * 17) % high for i in range(batch)]


# Inputs -----------------------------------------------------------------------------------


def _inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=DEVICE)  # noqa: E731
    uniform = lambda *shape: torch.rand(shape, generator=gen, device=DEVICE)  # noqa: E731
    if case["kind"] == "gated":
        rows, width = case["rows"], case["width"]
        # The gate is the second half of a projection's rows, as the layer made them.
        return dict(x=normal(rows, width).to(BF16), gate=normal(rows, 2 * width).to(BF16)[:, width:],
                    weight=(1 + 0.1 * normal(case["group"])).to(BF16))
    if case["kind"] == "block":
        rows, hidden = case["rows"], case["hidden"]
        gate = None if case["gate"] == "none" else normal(*(() if case["gate"] == "hidden" else (rows,)), hidden)
        return dict(x=(3 * normal(rows, hidden)).to(BF16), block=normal(rows, hidden).to(BF16),
                    gate=None if gate is None else gate.to(BF16), pre=(1 + 0.1 * normal(hidden)).to(BF16),
                    post=(1 + 0.1 * normal(hidden)).to(BF16) if case["post"] else None)
    lengths = _lengths(case)
    n, heads, groups, dk, dv = sum(lengths), case["heads"], case["key_heads"], case["key_dim"], case["value_dim"]
    ends = (groups * dk, 2 * groups * dk, 2 * groups * dk + heads * dv)
    rows = normal(n, ends[2]).to(BF16)
    rows[:, ends[0] : ends[1]] *= dk ** -0.5   # keys of about unit length
    q, k, v = rows[:, : ends[0]], rows[:, ends[0] : ends[1]], rows[:, ends[1] :]
    if not case["fused"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    made = dict(q=q.unflatten(1, (groups, dk)), k=k.unflatten(1, (groups, dk)), v=v.unflatten(1, (heads, dv)),
                lengths=lengths, decay=None, log_decay=None, strengths=None)
    # Rates of 1 to 16 and time steps about 0.001 to 0.1, as such layers begin and stay near.
    step = torch.nn.functional.softplus(
        torch.log(torch.expm1(torch.exp(uniform(heads) * math.log(100.0)) * 1e-3)) + 0.5 * normal(n, heads))
    if case["decay"] == "head":
        made["decay"] = -torch.exp2(-8.0 * torch.arange(1, heads + 1, device=DEVICE) / heads)
    else:
        made["log_decay"] = -(1 + 15 * uniform(heads)) * step
    if case["strengths"]:
        made["strengths"] = step
    # One state more than sequences, taken in another order than the batch's.
    made["states"] = normal(case["batch"] + 1, heads, dk, dv) * 0.5
    made["slots"] = torch.randperm(case["batch"] + 1, generator=torch.Generator().manual_seed(seed))[
        : case["batch"]].tolist()
    return made


class _Leaf:
    """A norm's weight and epsilon, as a block declares it."""

    def __init__(self, weight: torch.Tensor) -> None:
        self.weight, self.eps = weight, EPS


def prepare(case: dict, seed: int) -> dict:
    state = dict(_inputs(case, seed), case=case)
    if own:
        import __graft_entry__

        __graft_entry__.load_package()
        if case["kind"] == "gated":
            from mlx_omnia_amd.kernels.gated_norm import GatedRmsNorm

            state["norm"] = GatedRmsNorm(_Leaf(state["weight"]), activation=case["act"],
                                         gate_first=case["gate_first"])
        elif case["kind"] == "block":
            from mlx_omnia_amd.kernels.block_norm import BlockNorm

            state["norm"] = BlockNorm(_Leaf(state["pre"]), None if state["post"] is None else _Leaf(state["post"]),
                                      residual_scale=case["residual_scale"], block_scale=case["block_scale"],
                                      activation="sigmoid")
        else:
            from mlx_omnia_amd.kernels.linear_attention import LinearAttention, LinearBatch

            state["batch"] = LinearBatch(state["slots"], state["lengths"], device=DEVICE)
            state["mixer"] = LinearAttention(
                state["states"], heads=case["heads"], key_heads=case["key_heads"], key_dim=case["key_dim"],
                value_dim=case["value_dim"], scale=case["key_dim"] ** -0.5, dtype=BF16, decay=state["decay"])
    elif case["kind"] == "mix":
        state.update(_chunks(state))
    return state


def run(state: dict):
    case = state["case"]
    if not own:
        return {"mix": _plain_mix, "gated": _plain_gated, "block": _plain_block}[case["kind"]](state)
    if case["kind"] == "gated":
        return state["norm"](state["x"], state["gate"])
    if case["kind"] == "block":
        return state["norm"](state["x"], state["block"], state["gate"])
    context = state["mixer"](state["batch"], state["q"], state["k"], state["v"], state["log_decay"],
                             state["strengths"])
    return context, state["states"]


# The plain form ---------------------------------------------------------------------------


def _chunks(state: dict) -> dict:
    """The tokens of each chunk [chunks, width], -1 past its end, whose sequence it is of, and
    the last chunk of each sequence."""
    lengths = torch.tensor(state["lengths"], device=DEVICE)
    width = min(CHUNK, max(state["lengths"]))
    count = (lengths + width - 1) // width
    whose = torch.repeat_interleave(torch.arange(len(lengths), device=DEVICE), count)
    which = torch.arange(len(whose), device=DEVICE) - (torch.cumsum(count, 0) - count)[whose]
    at = which[:, None] * width + torch.arange(width, device=DEVICE)
    tokens = (torch.cumsum(lengths, 0) - lengths)[whose][:, None] + at
    return dict(tokens=torch.where(at < lengths[whose][:, None], tokens, -1), whose=whose,
                last=torch.cumsum(count, 0) - 1, index=torch.tensor(state["slots"], device=DEVICE))


def _plain_mix(state: dict):
    case = state["case"]
    heads, group = case["heads"], case["heads"] // case["key_heads"]
    tokens, whose, last = state["tokens"], state["whose"], state["last"]
    chunks, width = tokens.shape
    there = (tokens >= 0)[:, None]                                    # [chunks, 1, width]
    held = tokens.clamp(min=0)
    pick = lambda x: x[held].transpose(1, 2).to(F32) * there[..., None]  # noqa: E731 [chunks, heads, width, d]
    q = pick(state["q"]).repeat_interleave(group, dim=1)
    k = pick(state["k"]).repeat_interleave(group, dim=1)
    v = pick(state["v"])
    if state["log_decay"] is None:
        gates = state["decay"].to(F64)[None, :, None].expand(chunks, heads, width) * there
    else:
        gates = state["log_decay"][held].transpose(1, 2).to(F64) * there
    if state["strengths"] is not None:
        v = v * state["strengths"][held].transpose(1, 2)[..., None]
    to = torch.cumsum(gates, dim=2)                                   # in 64 bits: its differences count
    seen = torch.ones(width, width, dtype=torch.bool, device=DEVICE).tril()
    between = torch.exp(torch.where(seen, to[..., :, None] - to[..., None, :], -math.inf).to(F32))
    whole = to[..., -1]                                               # [chunks, heads]
    new = torch.matmul((k * torch.exp(whole[..., None] - to).to(F32)[..., None]).transpose(2, 3).contiguous(), v)
    # Each chunk's first state: the sequence's, and what its earlier chunks have added, decayed.
    behind = torch.cumsum(whole, dim=0)
    before = behind - whole
    earlier = (whose[:, None] == whose[None]) & torch.ones(chunks, chunks, dtype=torch.bool, device=DEVICE).tril(-1)
    carry = torch.where(earlier, before.t()[:, :, None] - behind.t()[:, None], -math.inf)
    held_states = state["states"][state["index"]]
    opened = before[(last - torch.bincount(whose, minlength=len(last)) + 1)][whose]
    first = torch.matmul(torch.exp(carry.to(F32)), new.transpose(0, 1).flatten(2)).unflatten(
        2, new.shape[2:]).transpose(0, 1)
    first = first + torch.exp(before - opened).to(F32)[..., None, None] * held_states[whose]
    context = torch.matmul(q, first) * torch.exp(to).to(F32)[..., None]
    context = context + torch.matmul(torch.matmul(q, k.transpose(2, 3).contiguous()) * between, v)
    context = context * case["key_dim"] ** -0.5
    state["states"][state["index"]] = (first * torch.exp(whole).to(F32)[..., None, None] + new)[last]
    return context.transpose(1, 2)[tokens >= 0].to(BF16), state["states"]


def _act(x: torch.Tensor, name: str) -> torch.Tensor:
    gate = 1 / (1 + torch.exp(-x))
    return x * gate if name == "silu" else gate


def _norm(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * weight


def _plain_gated(state: dict):
    case, shape = state["case"], (-1, state["case"]["group"])
    x, gate = (state[name].to(F32).unflatten(1, shape) for name in ("x", "gate"))
    weight, gate = state["weight"].to(F32), _act(gate, case["act"])
    y = _norm(x * gate, weight) if case["gate_first"] else _norm(x, weight) * gate
    return y.flatten(1).to(BF16)


def _plain_block(state: dict):
    case, block = state["case"], state["block"].to(F32)
    if state["post"] is not None:
        block = _norm(block, state["post"].to(F32))
    if state["gate"] is not None:
        block = block * _act(state["gate"].to(F32), "sigmoid")
    total = case["residual_scale"] * state["x"].to(F32) + case["block_scale"] * block
    return total.to(BF16), _norm(total, state["pre"].to(F32)).to(BF16)


# What a pass cannot do without ------------------------------------------------------------


def work(case: dict) -> dict:
    if case["kind"] == "gated":
        n = case["rows"] * case["width"]
        return dict(bytes=6 * n + 2 * case["group"], flops=10 * n)
    if case["kind"] == "block":
        n, hidden = case["rows"] * case["hidden"], case["hidden"]
        gate = {"none": 0, "hidden": hidden, "rows": n}[case["gate"]]
        return dict(bytes=2 * (4 * n + gate + hidden * (1 + case["post"])), flops=12 * n)
    n, heads, keys = sum(_lengths(case)), case["heads"], case["key_heads"]
    dk, dv = case["key_dim"], case["value_dim"]
    gates = 4 * n * heads * ((case["decay"] == "token") + case["strengths"])
    return dict(bytes=2 * n * (2 * keys * dk + 2 * heads * dv) + gates + 8 * case["batch"] * heads * dk * dv,
                flops=4 * n * heads * dk * dv)


# The same in 64 bits ----------------------------------------------------------------------


def exact(case: dict, seed: int):
    inputs = _inputs(case, seed)
    wide = {name: x.to(F64) for name, x in inputs.items() if isinstance(x, torch.Tensor)}
    if case["kind"] == "gated":
        x, z = (wide[name].reshape(case["rows"], -1, case["group"]) for name in ("x", "gate"))
        z = torch.sigmoid(z) * (z if case["act"] == "silu" else 1)
        y = x * z if case["gate_first"] else x
        y = y / torch.sqrt(y.square().sum(dim=-1, keepdim=True) / case["group"] + EPS)
        y = y * wide["weight"]
        return (y if case["gate_first"] else y * z).reshape(case["rows"], -1)
    if case["kind"] == "block":
        hidden, y = case["hidden"], wide["block"]
        if "post" in wide:
            y = wide["post"] * y / torch.sqrt(y.square().sum(dim=-1, keepdim=True) / hidden + EPS)
        if "gate" in wide:
            y = y * torch.sigmoid(wide["gate"])
        s = wide["x"] * case["residual_scale"] + y * case["block_scale"]
        return s, wide["pre"] * s / torch.sqrt(s.square().sum(dim=-1, keepdim=True) / hidden + EPS)
    # The sum over all earlier tokens, as the recurrence unrolls to; a block of queries at a time.
    group, states, n = case["heads"] // case["key_heads"], wide["states"], sum(inputs["lengths"])
    gates = wide["log_decay"] if "log_decay" in wide else wide["decay"].expand(n, -1)
    values = wide["v"] * wide["strengths"][..., None] if "strengths" in wide else wide["v"]
    context = torch.empty_like(wide["v"])
    if case["tokens"] == 1:
        index = torch.tensor(inputs["slots"], device=DEVICE)
        q, k = (wide[name].repeat_interleave(group, dim=1) for name in ("q", "k"))
        now = states[index] * torch.exp(gates)[..., None, None] + k[..., None] * values[..., None, :]
        states[index] = now
        return (q[..., None] * now).sum(dim=2) / math.sqrt(case["key_dim"]), states
    first = 0
    for slot, count in zip(inputs["slots"], inputs["lengths"]):
        mine = slice(first, first + count)
        to = torch.cumsum(gates[mine], dim=0).t().contiguous()        # [heads, count]
        step = max(1, min(count, (1 << 25) // count))
        for h in range(case["heads"]):
            q, k, v, g = wide["q"][mine, h // group], wide["k"][mine, h // group], values[mine, h], to[h]
            for low in range(0, count, step):
                high = min(count, low + step)
                apart = g[low:high, None] - g[None, :high]
                apart.masked_fill_(torch.arange(high, device=DEVICE)[None] > torch.arange(
                    low, high, device=DEVICE)[:, None], -math.inf)
                weight = torch.mm(q[low:high], k[:high].t().contiguous()) * apart.exp_()
                mixed = torch.mm(weight, v[:high].contiguous())
                mixed += torch.exp(g[low:high, None]) * torch.mm(q[low:high], states[slot, h])
                context[first + low : first + high, h] = mixed / math.sqrt(case["key_dim"])
            left = torch.exp(g[-1] - g)[:, None] * k
            states[slot, h] = states[slot, h] * torch.exp(g[-1]) + torch.mm(left.t().contiguous(), v.contiguous())
        first += count
    return context, states
