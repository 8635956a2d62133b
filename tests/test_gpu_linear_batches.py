"""What a batch of the linear attention holds, and what its first call waits for."""

from __future__ import annotations

import gc
import weakref

import pytest
import torch

from linear_cases import check, inputs
from mlx_omnia_amd.kernels.linear_attention import HipLinearAttention, LinearAttention, LinearBatch

pytestmark = pytest.mark.gpu


def layer(states, key_heads):
    _, heads, key_dim, value_dim = states.shape
    mixer = LinearAttention(states, heads=heads, key_heads=key_heads, key_dim=key_dim, value_dim=value_dim,
                            scale=key_dim ** -0.5, dtype=torch.bfloat16)
    assert isinstance(mixer.strategy, HipLinearAttention)
    return mixer


@pytest.mark.parametrize("tokens", [[1, 3], [200, 1]])
def test_a_batch_keeps_no_layer_alive(tokens):
    made, _, states, slots = inputs(tokens, 4, 2, 64, 64, device="cuda")
    batch, kept = LinearBatch(slots, tokens), layer(states.clone(), 2)
    kept(batch, **made)
    gc.collect()
    before = torch.cuda.memory_allocated()
    mixer = layer(states.clone(), 2)
    mixer(batch, **made)
    gone = weakref.ref(mixer.strategy)
    del mixer
    gc.collect()
    assert gone() is None and torch.cuda.memory_allocated() == before
    own = kept.strategy.core.states
    before = own.clone()
    check(kept(batch, **made), own, made, None, before, slots, tokens, 0.125)


@pytest.mark.parametrize("tokens", [[1, 1, 1], [300, 1, 70], [2000]])
@pytest.mark.parametrize("own", [False, True])
def test_a_first_call_does_not_wait_for_earlier_work(tokens, own):
    """Its lists go up while the caller's stream is busy: the host is back before that is done."""
    made, _, states, slots = inputs(tokens, 4, 2, 64, 64, device="cuda")
    mixer, before = layer(states, 2), states.clone()
    warm = layer(states.clone(), 2)
    warm(LinearBatch(slots, tokens), **made)   # what a process does once
    wide = torch.randn(8192, 8192, device="cuda")
    torch.mm(wide, wide)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream() if own else torch.cuda.current_stream()
    with torch.cuda.stream(stream):
        for _ in range(8):   # tens of milliseconds
            torch.mm(wide, wide)
        earlier = torch.cuda.Event()
        earlier.record(stream)
        out = mixer(LinearBatch(slots, tokens), **made)
        busy = not earlier.query()
    stream.synchronize()
    assert busy
    check(out, states, made, None, before, slots, tokens, 0.125)


@pytest.mark.parametrize("own", [False, True])
def test_a_dropped_batch_is_read_before_another_takes_its_place(own):
    """Lists of batches that are made and dropped while the stream that reads them is behind."""
    tokens = [130, 1, 1]
    made, _, states, slots = inputs(tokens, 4, 2, 64, 64, device="cuda")
    mixer = layer(states, 2)
    wide = torch.randn(8192, 8192, device="cuda")
    mixer(LinearBatch(slots, tokens), **made)
    torch.mm(wide, wide)
    torch.cuda.synchronize()
    want, stream = states.clone(), torch.cuda.Stream() if own else torch.cuda.current_stream()
    reference, turns = layer(want, 2), [slots, slots[::-1], slots[1:] + slots[:1]]
    for turn in turns:
        kept = LinearBatch(turn, tokens)
        reference(kept, **made)
        torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(8):   # tens of milliseconds
            torch.mm(wide, wide)
        earlier = torch.cuda.Event()
        earlier.record(stream)
        for turn in turns:
            batch = LinearBatch(turn, tokens)
            mixer(batch, **made)
            del batch
        busy = not earlier.query()
    stream.synchronize()
    assert busy and torch.equal(states, want)


@pytest.mark.parametrize("tokens", [[1, 1, 1], [300, 1, 70]])
def test_a_call_on_another_stream_waits_for_the_lists(tokens):
    """The first call stands behind other work on its stream; another layer's, on a stream that waits for none of
    that, reads the same lists."""
    made, _, first, slots = inputs(tokens, 4, 2, 64, 64, device="cuda")
    second = first.flip(0).contiguous()
    pools = [first.clone(), second.clone()]
    mixers, wide = [layer(p, 2) for p in pools], torch.randn(8192, 8192, device="cuda")
    for mixer in mixers:   # what a process does once
        mixer(LinearBatch([s for s in range(len(first)) if s not in slots][:1], [0]), **{k: None if t is None else t[:0] for k, t in made.items()})
    torch.mm(wide, wide)
    streams = [torch.cuda.Stream() for _ in pools]
    torch.cuda.synchronize()
    batch, outs = LinearBatch(slots, tokens), []
    with torch.cuda.stream(streams[0]):
        for _ in range(8):   # tens of milliseconds
            torch.mm(wide, wide)
        earlier = torch.cuda.Event()
        earlier.record()
    for mixer, stream in zip(mixers, streams):
        with torch.cuda.stream(stream):
            outs.append(mixer(batch, **made))
    busy = not earlier.query()
    torch.cuda.synchronize()
    assert busy
    for out, pool, before in zip(outs, pools, (first, second)):
        check(out, pool, made, None, before, slots, tokens, 0.125)


def test_under_another_default_device():
    """A batch is made and first called where tensors are made on the GPU by default."""
    made, _, states, slots = inputs([70, 1], 4, 2, 64, 64, device="cuda")
    before = states.clone()
    with torch.device("cuda"):
        out = layer(states, 2)(LinearBatch(slots, [70, 1]), **made)
    check(out, states, made, None, before, slots, [70, 1], 0.125)
