"""HIP linear attention against the float64 oracle: every geometry, lengths around the ends of what
the kernels take together, mixed batches, strides, decays and values at the edge, streams, graphs,
and a layer's run from the gate to the next block's norm."""

from __future__ import annotations

import math

import pytest
import torch

from linear_cases import check, inputs
from mlx_omnia_amd.kernels.block_norm import BlockNorm, HipBlockNorm
from mlx_omnia_amd.kernels.gate_softplus import GateSoftplus
from mlx_omnia_amd.kernels.gated_norm import GatedRmsNorm, HipGatedRmsNorm
from mlx_omnia_amd.kernels.leaf import RMSNormLeaf
from mlx_omnia_amd.kernels import linear_attention
from mlx_omnia_amd.kernels.linear_attention import HipLinearAttention, LinearAttention, LinearBatch
from mlx_omnia_amd.kernels.resolve import FALLBACKS

pytestmark = pytest.mark.gpu


def layer(states, key_heads, decay=None, **more):
    _, heads, key_dim, value_dim = states.shape
    mixer = LinearAttention(states, heads=heads, key_heads=key_heads, key_dim=key_dim, value_dim=value_dim,
                            scale=key_dim ** -0.5, dtype=torch.bfloat16, decay=decay, **more)
    assert more or isinstance(mixer.strategy, HipLinearAttention)
    return mixer


def run(tokens, heads, key_heads, key_dim, value_dim, **kind):
    print(f"linear_attention tokens={tokens} heads={heads}/{key_heads} dims={key_dim}x{value_dim} {kind}", flush=True)
    made, fixed, states, slots = inputs(tokens, heads, key_heads, key_dim, value_dim, device="cuda", **kind)
    before = states.clone()
    out = layer(states, key_heads, fixed)(LinearBatch(slots, tokens), **made)
    torch.cuda.synchronize()
    check(out, states, made, fixed, before, slots, tokens, key_dim ** -0.5)
    rest = [s for s in range(len(states)) if s not in slots or tokens[slots.index(s)] == 0]
    assert torch.equal(states[rest], before[rest])


@pytest.mark.parametrize("key_dim", [64, 128])
@pytest.mark.parametrize("value_dim", [64, 128])
@pytest.mark.parametrize("tokens", [[1], [1, 1, 1, 1, 1], [2], [31], [64], [65], [128], [200], [3, 0, 1, 70, 1]])
def test_against_the_oracle(key_dim, value_dim, tokens):
    run(tokens, 4, 2, key_dim, value_dim, seed=len(tokens))


@pytest.mark.parametrize("count", [15, 16, 17, 32, 33, 63, 95, 127, 129, 192, 193, 257, 511, 1025])
def test_lengths(count):
    run([count], 2, 2, 128, 128, seed=count, strengths=count % 2 == 0)


@pytest.mark.parametrize("heads,key_heads", [(1, 1), (8, 1), (12, 4), (3, 3), (64, 2)])
@pytest.mark.parametrize("decay", ["token", "head"])
@pytest.mark.parametrize("strengths", [False, True])
def test_heads_and_gates(heads, key_heads, decay, strengths):
    run([1, 77], heads, key_heads, 128, 64, decay=decay, strengths=strengths, fused=True)


GEOMETRIES = [(2, 2, 128, 128), (2, 1, 64, 128), (3, 3, 128, 64), (4, 2, 128, 64), (4, 1, 128, 64), (8, 1, 64, 64),
              (6, 3, 64, 64), (1, 1, 64, 64)]


@pytest.mark.parametrize("size", [1, 2, 5])
@pytest.mark.parametrize("heads,key_heads,key_dim,value_dim", GEOMETRIES)
def test_in_pieces(monkeypatch, size, heads, key_heads, key_dim, value_dim):
    """Pieces of so many chunks: sequences of one, two, three and many, whatever the plan would do."""
    monkeypatch.setattr(linear_attention, "piece_chunks", lambda chunks, places: size)
    run([700, 2, 129, 64, 65, 0, 300], heads, key_heads, key_dim, value_dim, strengths=True, fused=True)


@pytest.mark.parametrize("where", ["values", "keys", "strengths", "log_decay"])
@pytest.mark.parametrize("at", [0, 63, 200, 449])
def test_in_pieces_what_is_not_finite_stays_with_later_tokens(monkeypatch, where, at):
    monkeypatch.setattr(linear_attention, "piece_chunks", lambda chunks, places: 2)
    made, _, states, slots = inputs([450], 4, 1, 128, 64, device="cuda", strengths=True)
    plain, _, clean, _ = inputs([450], 4, 1, 128, 64, device="cuda", strengths=True)
    made[where].reshape(450, -1)[at, 5 if where in ("values", "keys") else 1] = math.nan
    out = layer(states, 1)(LinearBatch(slots, [450]), **made)
    want = layer(clean, 1)(LinearBatch(slots, [450]), **plain)
    assert torch.isfinite(out[:at]).all()
    torch.testing.assert_close(out[:at].float(), want[:at].float(), rtol=2 ** -7, atol=2 ** -10)
    head, columns = (0, slice(5, 6)) if where == "values" else (slice(None), slice(None)) if where == "keys" else (
        1, slice(None))
    assert not torch.isfinite(out[at:, head, columns]).any() and not torch.isfinite(out[449, head, columns]).any()
    state = states[slots[0]]
    assert not torch.isfinite(state[head, 5 if where == "keys" else slice(None), columns]).any()
    if where != "keys":
        other = torch.ones_like(out, dtype=torch.bool)
        other[:, head, columns] = False
        assert torch.isfinite(out[other]).all()


def test_far_offsets():
    """States past 2^31 elements and 2^33 bytes from the first, rows 2^23 elements apart."""
    heads, d, tokens = 8, 64, [70, 1]
    made, _, small, slots = inputs(tokens, heads, 2, d, d, device="cuda", slots=4, strengths=True)
    before = small.clone()
    want = layer(small, 2)(LinearBatch(slots, tokens), **made)
    pool = torch.empty(70000, heads, d, d, device="cuda")   # 9.2 GB
    far = [69999 - s for s in slots]
    pool[far] = before[slots]
    wide = torch.empty(71, 1 << 23, dtype=torch.bfloat16, device="cuda")   # 1.2 GB, 0.6 G elements
    rows = {name: torch.as_strided(wide, t.shape, (1 << 23, t.shape[2], 1), 1 << 12).copy_(t)
            for name, t in (("queries", made["queries"]),)}
    got = layer(pool, 2)(LinearBatch(far, tokens), **{**made, **rows})
    assert torch.equal(got, want) and torch.equal(pool[far], small[slots])


def test_sequences_of_all_lengths():
    run([300, 1, 64, 7, 0, 129, 1, 1, 63, 500], 4, 2, 128, 128, fused=True, strengths=True)


def test_a_long_sequence():
    """Enough of one for its work to be cut into pieces, and slow decays, which carry over all of them."""
    made, _, states, slots = inputs([4500], 2, 1, 128, 128, device="cuda")
    made["log_decay"] = made["log_decay"] * 1e-3
    before = states.clone()
    out = layer(states, 1)(LinearBatch(slots, [4500]), **made)
    check(out, states, made, None, before, slots, [4500], 128 ** -0.5)


def test_fast_decays_before_slow_ones():
    """The sums of a hundred fast decays and a slow one differ by the slow one: none of it may be lost."""
    made, _, states, slots = inputs([150], 4, 2, 128, 128, device="cuda")
    fast = torch.arange(150, device="cuda") % 64 < 40
    made["log_decay"] = torch.where(fast[:, None], -30.0, -1e-3) * torch.ones(1, 4, device="cuda")
    before = states.clone()
    out = layer(states, 2)(LinearBatch(slots, [150]), **made)
    check(out, states, made, None, before, slots, [150], 128 ** -0.5)


@pytest.mark.parametrize("decay", [0.0, -0.0, -1e-30, -88.0, -104.0, -3e38, -math.inf])
@pytest.mark.parametrize("tokens", [1, 100])
def test_decays_at_the_edge(decay, tokens):
    made, _, states, slots = inputs([tokens], 2, 2, 64, 64, device="cuda")
    made["log_decay"][::3] = decay
    before = states.clone()
    out = layer(states, 2)(LinearBatch(slots, [tokens]), **made)
    assert torch.isfinite(out).all()
    check(out, states, made, None, before, slots, [tokens], 0.125)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("where", ["values", "keys", "queries", "strengths", "log_decay"])
@pytest.mark.parametrize("at", [0, 37, 64, 129])
def test_what_is_not_finite_stays_with_later_tokens(bad, where, at):
    if where == "log_decay" and bad == -math.inf:
        pytest.skip("a decay to nothing, tested above")
    made, _, states, slots = inputs([130, 1], 2, 1, 128, 128, device="cuda", strengths=True)
    plain, _, clean, _ = inputs([130, 1], 2, 1, 128, 128, device="cuda", strengths=True)
    made[where].reshape(131, -1)[at, 5 if where not in ("strengths", "log_decay") else 1] = bad
    out = layer(states, 1)(LinearBatch(slots, [130, 1]), **made)
    want = layer(clean, 1)(LinearBatch(slots, [130, 1]), **plain)
    assert torch.isfinite(out[:at]).all() and torch.isfinite(out[130]).all()
    # The tokens before it, the other sequence's, and the columns of v that have no part in it.
    torch.testing.assert_close(out[:at].float(), want[:at].float(), rtol=2 ** -7, atol=2 ** -10)
    assert torch.equal(out[130], want[130]) and torch.equal(states[slots[1]], clean[slots[1]])
    if where == "values":
        assert not torch.isfinite(out[at:130, 0, 5]).any()
        assert torch.isfinite(out[:, :, 6:]).all() and torch.isfinite(out[:, 1]).all()
    elif where == "queries":
        assert not torch.isfinite(out[at]).any() and torch.isfinite(out[at + 1 :]).all()
        assert torch.isfinite(states).all()
    else:
        assert not torch.isfinite(out[129 if where == "keys" else at, 1]).any()


def test_a_call_continues_where_one_ended():
    made, _, states, slots = inputs([200], 4, 2, 128, 128, device="cuda")
    before, mixer = states.clone(), layer(states, 2)
    outs = [mixer(LinearBatch(slots, [n]), **{k: None if t is None else t[a : a + n] for k, t in made.items()})
            for a, n in ((0, 1), (1, 100), (101, 1), (102, 1), (103, 97))]
    check(torch.cat(outs), states, made, None, before, slots, [200], 128 ** -0.5)


def test_rows_that_lie_otherwise():
    """Heads apart, unaligned rows, transposed gates: copied or read as they are, with the same results."""
    tokens = [1, 90]
    made, _, states, slots = inputs(tokens, 4, 2, 64, 128, device="cuda", strengths=True)
    clean, batch = states.clone(), LinearBatch(slots, tokens)
    want = layer(clean, 2)(batch, **made)
    apart = {name: torch.empty(t.shape[1], t.shape[0], t.shape[2], dtype=t.dtype, device="cuda").transpose(0, 1).copy_(t)
             for name, t in made.items() if t.dim() == 3}
    odd = {name: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)
           for name, t in made.items()}
    turned = {name: t.t().contiguous().t() for name, t in made.items() if t.dim() == 2}
    for change in (apart, odd, turned):
        pool = states.clone()
        got = layer(pool, 2)(batch, **{**made, **change})
        assert torch.equal(got, want) and torch.equal(pool, clean)


def test_same_inputs_same_bits():
    made, _, states, slots = inputs([700, 3, 1], 8, 4, 128, 128, device="cuda")
    first = None
    for _ in range(3):
        pool = states.clone()
        got = layer(pool, 4)(LinearBatch(slots, [700, 3, 1]), **made), pool
        assert first is None or all(torch.equal(a, b) for a, b in zip(got, first))
        first = got


def test_on_another_stream():
    made, _, states, slots = inputs([300, 1], 4, 2, 128, 128, device="cuda")
    clean, batch = states.clone(), LinearBatch(slots, [300, 1])
    want = layer(clean, 2)(batch, **made)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = layer(states, 2)(batch, **made)
    stream.synchronize()
    assert torch.equal(got, want) and torch.equal(states, clean)


@pytest.mark.parametrize("tokens", [[1, 2], [0, 0], [], [600, 65]])
def test_any_batch_on_another_stream_than_its_lists(tokens):
    made, _, states, slots = inputs(tokens, 4, 2, 64, 64, device="cuda")
    clean, batch = states.clone(), LinearBatch(slots, tokens)
    want = layer(clean, 2)(batch, **made)   # lays the lists out here
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = layer(states, 2)(batch, **made)
    stream.synchronize()
    assert torch.equal(got, want) and torch.equal(states, clean)


def test_two_layers_take_one_batch_at_once():
    """Each call has a workspace of its own."""
    tokens = [2000, 1, 300]
    made, _, first, slots = inputs(tokens, 4, 2, 128, 64, device="cuda")
    second = first.flip(0).contiguous()
    pools, batch = [first, second], LinearBatch(slots, tokens)
    clean = [p.clone() for p in pools]
    want = [layer(p, 2)(batch, **made) for p in clean]
    mixers, streams = [layer(p, 2) for p in pools], [torch.cuda.Stream() for _ in pools]
    got = []
    for mixer, stream in zip(mixers, streams):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got.append(mixer(batch, **made))
    torch.cuda.synchronize()
    for a, b in zip(got + pools, want + clean):
        assert torch.equal(a, b)


def test_a_batch_dropped_under_way_on_another_stream():
    """Its lists' memory is nobody else's before the call has read them."""
    made, _, states, slots = inputs([300, 1], 4, 2, 128, 128, device="cuda")
    mixer, batch = layer(states, 2), LinearBatch(slots, [300, 1])
    mixer(batch, **made)   # lays the lists out here
    lists = next(iter(batch._lists.values()))
    at, stream = lists.runs.untyped_storage().data_ptr(), torch.cuda.Stream()
    wide = torch.randn(8192, 8192, device="cuda")
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(8):   # tens of milliseconds
            torch.mm(wide, wide)
        mixer(batch, **made)
    del batch, lists
    others = [torch.empty(64, dtype=torch.int32, device="cuda") for _ in range(64)]
    busy = not stream.query()
    held = {t.data_ptr() for t in others}
    stream.synchronize()
    assert busy and at not in held


@pytest.mark.parametrize("tokens", [[1, 1, 1], [150, 1]])
def test_captured_and_replayed(tokens):
    made, _, states, slots = inputs(tokens, 4, 2, 128, 128, device="cuda")
    batch, mixer = LinearBatch(slots, tokens), layer(states, 2)
    eager = states.clone()
    other = layer(eager, 2)
    with pytest.raises((ValueError, RuntimeError)), torch.cuda.graph(torch.cuda.CUDAGraph()):
        mixer(batch, **made)
    torch.cuda.synchronize()
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        mixer(batch, **made)
    torch.cuda.current_stream().wait_stream(warm)
    other(batch, **made)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mixer(batch, **made)
    for step in range(4):
        for t in (made["queries"], made["keys"], made["values"]):
            t.copy_(torch.randn_like(t))
        graph.replay()
        want = other(batch, **made)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(states, eager), step


def test_followed_calls_and_other_types_run_in_torch():
    made, _, states, slots = inputs([5], 4, 2, 64, 64, device="cuda")
    batch, before = LinearBatch(slots, [5]), dict(FALLBACKS)
    leaf = made["values"].detach().clone().requires_grad_()
    out = layer(states, 2)(batch, **{**made, "values": leaf})
    out.float().sum().backward()
    assert torch.isfinite(leaf.grad).all()
    assert FALLBACKS["HipLinearAttention -> DefaultLinearAttention"] == before.get(
        "HipLinearAttention -> DefaultLinearAttention", 0) + 1


def test_many_batches_over_the_same_pool():
    """Slots in turn, a fork's copy and a fresh one's zeros between calls, on one stream."""
    heads, d = 4, 64
    made, _, states, _ = inputs([200], heads, 2, d, d, device="cuda", slots=6)
    other, mixer = states.clone(), layer(states, 2)
    reference = layer(other, 2, reference=True)
    for slots, tokens in (([0, 3], [100, 1]), ([3, 5], [1, 1]), ([1, 0], [64, 65]), ([2], [200]), ([0, 1, 2], [3, 4, 5])):
        n = sum(tokens)
        part = {k: None if t is None else t[:n] for k, t in made.items()}
        for pool in (states, other):
            pool[4].zero_()
            pool[5] = pool[0]
        batch = LinearBatch(slots, tokens)
        got, want = mixer(batch, **part), reference(batch, **part)
        torch.testing.assert_close(got.float(), want.float(), rtol=2 ** -7, atol=2 ** -8)
        torch.testing.assert_close(states, other, rtol=2 ** -14, atol=2 ** -14)


def test_refusals():
    made, _, states, slots = inputs([5], 4, 2, 64, 64, device="cuda")
    mixer, batch = layer(states, 2), LinearBatch(slots, [5])
    for change in (dict(queries=made["queries"].float()), dict(keys=made["keys"].cpu()),
                   dict(log_decay=made["log_decay"].bfloat16()), dict(strengths=torch.ones(5, 4)), dict(log_decay=None),
                   dict(queries=made["queries"][:4]), dict(values=made["values"][:, :2]),
                   dict(log_decay=made["log_decay"][0]), dict(strengths=torch.ones(4, device="cuda"))):
        with pytest.raises(ValueError):
            mixer(batch, **{**made, **change})
    with pytest.raises(ValueError):
        mixer(LinearBatch([len(states)], [5]), **made)
    with pytest.raises(ValueError):
        mixer(LinearBatch(slots, [5], device="cpu"), **made)
    odd = LinearAttention(torch.zeros(2, 4, 96, 64, device="cuda"), heads=4, key_heads=2, key_dim=96, value_dim=64,
                          scale=1.0, dtype=torch.bfloat16)
    assert not isinstance(odd.strategy, HipLinearAttention)


@pytest.mark.parametrize("tokens", [[1, 1], [90, 1]])
def test_a_layer_from_the_gate_to_the_next_norm(tokens):
    """Gate, mixer, gated norm, projection and join, against the Core chains in 32 bits from the same
    bf16 tensors: each stage's result, where the chain hands on what the kernels gave."""
    heads, key_heads, d, hidden = 4, 2, 128, 256
    made, _, states, slots = inputs(tokens, heads, key_heads, d, d, device="cuda", fused=True)
    n, gen = sum(tokens), torch.Generator().manual_seed(5)
    normal = lambda *shape: torch.randn(shape, generator=gen).cuda()  # noqa: E731
    a, z = normal(n, heads).bfloat16(), normal(n, heads * d).bfloat16()
    a_log, bias = normal(heads) * 0.5, normal(heads) - 3
    down = (normal(heads * d, hidden) / 16).bfloat16()
    residual, pre, post = normal(n, hidden).bfloat16(), 1 + 0.1 * normal(hidden), 1 + 0.1 * normal(hidden)
    weight = (1 + 0.1 * normal(d)).bfloat16()
    batch, results, core_states = LinearBatch(slots, tokens), [], states.clone()
    for reference, pool in ((False, states), (True, core_states)):
        gate = GateSoftplus(a_log, bias, reference=reference)
        mixer = layer(pool, key_heads, **(dict(reference=True) if reference else {}))
        norm = GatedRmsNorm(RMSNormLeaf(weight), reference=reference)
        join = BlockNorm(RMSNormLeaf(pre.bfloat16()), RMSNormLeaf(post.bfloat16()), residual_scale=0.5, block_scale=0.25,
                         reference=reference)
        assert reference or isinstance(norm.strategy, HipGatedRmsNorm) and isinstance(join.strategy, HipBlockNorm)
        stage = results[0] if reference else None
        g = gate(a)
        made["log_decay"] = stage[0] if reference else g
        context = mixer(batch, **made)
        normed = norm(stage[1] if reference else context, z.unflatten(1, (heads, d)))
        block = (stage[2] if reference else normed).flatten(1) @ down
        results.append((g, context, normed, *join(residual, stage[5] if reference else block), block))
    torch.testing.assert_close(results[0][0], results[1][0], rtol=2 ** -17, atol=2 ** -17)
    for got, want in zip(results[0][1:5], results[1][1:5]):
        # Both sides round once: a step apart at most, and sums of two hundred terms below that.
        torch.testing.assert_close(got.float(), want.float(), rtol=2 ** -7, atol=2 ** -8)
    torch.testing.assert_close(states, core_states, rtol=2 ** -14, atol=2 ** -14)
