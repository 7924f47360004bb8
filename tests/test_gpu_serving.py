"""The operators of serving in 8 bits together on the GPU: eager, in captured
steps, and two models at once."""

from __future__ import annotations

import pytest
import torch

import cuda_force_amd as cf
from tests.chunk_util import CODES
from tests.serving_util import Layer, serve

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HELD = [None, *CODES]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
def test_a_run(dtype, held):
    serve(Layer("cuda", dtype, held))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("held", HELD)
def test_captured_steps(dtype, held):
    """Decoding steps replayed from a graph, with eager steps of the same layer
    between them, against a layer that only runs eagerly."""
    layer, twin = Layer("cuda", dtype, held), Layer("cuda", dtype, held)
    prompt = {0: 37, 1: 16, 2: 5, 3: 1}
    layer.run(prompt)
    twin.run(prompt)
    sequences = layer.ints(0, 1, 2, 3)
    starts = layer.ints(0, 1, 2, 3, 4)
    x = torch.zeros(4, layer.hidden, dtype=dtype, device="cuda")

    def step(of, tokens):
        slots = cf.cache_extend(of.counts, of.tables, of.lens, sequences, of.BLOCK)
        return of.step(tokens, slots.view(-1), starts)

    state = [t.clone() for t in (layer.counts, layer.tables, layer.lens)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(layer, x)
    torch.cuda.current_stream().wait_stream(side)
    for t, old in zip((layer.counts, layer.tables, layer.lens), state):
        t.copy_(old)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, y = step(layer, x)
    # Capturing runs nothing: the layer stands where its twin does.
    for i in range(20):
        tokens = layer.tokens(4)
        if i % 5 == 4:
            got = step(layer, tokens)
        else:
            x.copy_(tokens)
            graph.replay()
            got = out, y
        want = step(twin, tokens)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
    for a, b in zip((*layer.caches, *layer.scales, layer.lens), (*twin.caches, *twin.scales, twin.lens)):
        assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("held", HELD)
def test_two_streams(held):
    """Two layers on two streams at once, each against itself alone."""
    def run(layer, steps):
        got = []
        for new in steps:
            slots = torch.cat([layer.extend([s], n) for s, n in sorted(new.items())])
            got.append(layer.step(layer.tokens(len(slots)), slots, layer.starts(new)))
        return got

    steps = [{0: 200, 1: 90}, *[{0: 1, 1: 1, 2: 1}] * 6]
    alone = [run(Layer("cuda", torch.bfloat16, held, seed=s), steps) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    layers = [Layer("cuda", torch.bfloat16, held, seed=s) for s in (1, 2)]
    torch.cuda.synchronize()
    got = [[], []]
    for new in steps:
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i] += run(layers[i], [new])
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        for one, other in zip(a, b):
            assert torch.equal(one[0], other[0]) and torch.equal(one[1], other[1])
