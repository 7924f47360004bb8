"""Storing into a paged cache and reading back on the GPU: bit by bit what the
plain form stores."""

from __future__ import annotations

import pytest
import torch

import cuda_force_amd as cf
from cuda_force_amd.paged_cache import _read_reference, _write_reference
from tests import codes_util

pytestmark = pytest.mark.gpu
CODES = [torch.int8, torch.float8_e4m3fn]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def bits(t):
    return t.contiguous().cpu().view({1: torch.int8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def run(keys, values, slots, pages, block, held):
    """Written and read on both sides; the cache starts with other content."""
    heads, dim = keys.shape[1:]
    gen = torch.Generator().manual_seed(5)
    k = torch.randint(-100, 100, (pages, block, heads, dim), generator=gen).float().to(held)
    state = [k, k.flip(0).contiguous()]
    state += [torch.rand(pages, block, heads, generator=gen) for _ in range(2)] if held in CODES else [None, None]
    on_gpu = [None if t is None else t.cuda() for t in state]
    cf.cache_write(keys.cuda(), values.cuda(), *on_gpu[:2], slots.cuda(), *on_gpu[2:])
    _write_reference(keys, values, *state[:2], slots, *state[2:])
    for got, want in zip(on_gpu, state):
        if want is not None:
            assert torch.equal(bits(got), bits(want))
    dtypes = DTYPES if held in CODES else [held]
    for dtype in dtypes:
        got = cf.cache_read(*on_gpu[:2], slots.cuda(), *on_gpu[2:], dtype=dtype)
        want = _read_reference(*state[:2], slots, *state[2:], dtype)
        for x, y in zip(got, want):
            assert torch.equal(torch.isnan(x).cpu(), torch.isnan(y))
            assert torch.equal(bits(x.nan_to_num(1.0, float("inf"), -float("inf"))),
                               bits(y.nan_to_num(1.0, float("inf"), -float("inf"))))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", CODES)
def test_hard_rows(dtype, held):
    for cols in (8, 64, 100):
        x = codes_util.hard_rows(dtype, cols).view(24, 1, cols)
        run(x, -x.flip(0), torch.arange(24).flip(0), 7, 4, held)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", [None, *CODES])
@pytest.mark.parametrize("dim", [1, 3, 16, 64, 80, 96, 128, 256, 300, 1024, 1100, 4096, 4104])
def test_head_sizes(dtype, held, dim):
    x = torch.randn(37, 2, 2, dim).to(dtype)
    run(x[:, 0], x[:, 1], torch.randperm(48)[:37], 3, 16, held or dtype)


@pytest.mark.parametrize("held", [torch.bfloat16, *CODES])
@pytest.mark.parametrize("tokens", [1, 2, 63, 500, 513, 1025, 5000])
def test_numbers_of_tokens_and_slots_named_again(held, tokens):
    gen = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, 3, 2, 32, generator=gen).to(torch.bfloat16)
    slots = torch.randint(-3, tokens + 40, (tokens,), generator=gen)  # some twice, some out of range
    run(x[:, 0], x[:, 2], slots, (tokens + 31) // 16, 16, held)
    run(x[:, 0], x[:, 2], torch.full((tokens,), 7), (tokens + 31) // 16, 16, held)
    run(x[:, 0], x[:, 2], torch.arange(tokens), (tokens + 31) // 16, 16, held)


def test_more_tokens_than_a_round_of_workgroups_holds():
    gen = torch.Generator().manual_seed(1)
    tokens = 300_001
    x = torch.randn(tokens, 2, 1, 16, generator=gen).to(torch.bfloat16)
    slots = torch.randint(0, tokens, (tokens,), generator=gen)
    run(x[:, 0], x[:, 1], slots, (tokens + 15) // 16, 16, torch.int8)


@pytest.mark.parametrize("held", [torch.bfloat16, *CODES])
def test_strides_and_alignment(held):
    fused = torch.randn(40, 6, 64).to(torch.bfloat16)
    slots = torch.randperm(64)[:40]
    run(fused[:, 2:4], fused[:, 4:], slots, 4, 16, held)
    run(fused[:, 2:4, 1:33], fused[:, 4:, 3:35], slots, 4, 16, held)
    run(fused[:, 2:4, ::2], fused[:, 4:, ::2], slots, 4, 16, held)
    run(fused[:1, :2].expand(40, 2, 64), fused[:, 4:], slots, 4, 16, held)
    by_head = torch.randn(2, 40, 64).to(torch.bfloat16).transpose(0, 1)
    run(by_head, by_head, slots, 4, 16, held)


def test_caches_that_are_not_aligned():
    """Slices of a larger tensor, an element past an aligned place."""
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(20, 2, 64, generator=gen).to(torch.bfloat16)
    slots = torch.randperm(32, generator=gen)[:20]
    for held in CODES:
        sets = []
        for device in ("cpu", "cuda"):
            flat = [torch.zeros(2 * 16 * 2 * 64 + 1, dtype=torch.int8, device=device) for _ in range(2)]
            k, v = (f[1:].view(held).view(2, 16, 2, 64) for f in flat)
            scales = [torch.ones(2, 16, 2, device=device) for _ in range(2)]
            cf.cache_write(x.to(device), x.to(device), k, v, slots.to(device), *scales)
            sets.append([*flat, *scales, *cf.cache_read(k, v, slots.to(device), *scales)])
        for a, b in zip(*sets):
            assert torch.equal(bits(a), bits(b))


def test_graph_and_stream():
    x = torch.randn(50, 2, 2, 64).to(torch.bfloat16).cuda()
    k, v = (torch.zeros(4, 16, 2, 64, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(4, 16, 2, device="cuda") for _ in range(2))
    slots = torch.randperm(64)[:50].cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cf.cache_write(x[:, 0], x[:, 1], k, v, slots, ks, vs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cf.cache_write(x[:, 0], x[:, 1], k, v, slots, ks, vs)
        got = cf.cache_read(k, v, slots, ks, vs, dtype=torch.bfloat16)
    for seed in range(3):
        torch.manual_seed(seed)
        x.copy_(torch.randn_like(x))
        slots.copy_(torch.randperm(64)[:50])
        graph.replay()
        torch.cuda.synchronize()
        state = [torch.zeros(4, 16, 2, 64, dtype=torch.int8) for _ in range(2)] + [torch.ones(4, 16, 2) for _ in range(2)]
        _write_reference(x[:, 0].cpu(), x[:, 1].cpu(), *state[:2], slots.cpu(), *state[2:])
        for a, b in zip(got, _read_reference(*state[:2], slots.cpu(), *state[2:], torch.bfloat16)):
            assert torch.equal(bits(a), bits(b))


def test_one_place_for_keys_and_values_is_refused():
    x = torch.randn(4, 2, 64, device="cuda")
    slots = torch.arange(4, device="cuda")
    cache = torch.zeros(2, 4, 2, 64, device="cuda")
    with pytest.raises(ValueError):
        cf.cache_write(x, x, cache, cache, slots)
    with pytest.raises(RuntimeError):
        cf.cache_write(x, x, cache, cache.view(cache.shape), slots)
    codes = [torch.zeros(2, 4, 2, 64, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = torch.zeros(2, 4, 2, device="cuda")
    with pytest.raises(RuntimeError):
        cf.cache_write(x, x, *codes, slots, scales, scales.view(scales.shape))
    assert (cache == 0).all() and (scales == 0).all()
