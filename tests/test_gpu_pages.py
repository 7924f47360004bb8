"""Pages of a paged cache on the GPU against the plain loops, bit for bit."""

from __future__ import annotations

import pytest
import torch

import cuda_force_amd as cf
from cuda_force_amd import paged_cache as plain
from tests.pages_util import ints, same, state, to

pytestmark = pytest.mark.gpu


def both(kernel, form, arguments, extra=()):
    """The operator on GPU copies and the plain form on CPU copies: the same
    results, and the same state afterwards."""
    gpu, cpu = to("cuda", arguments), to("cpu", arguments)
    a, b = kernel(*gpu, *extra), form(*cpu, *extra)
    same([x for x in (a if isinstance(a, tuple) else (a,)) if x is not None],
         [x for x in (b if isinstance(b, tuple) else (b,)) if x is not None])
    same(gpu, cpu)
    return a


def random_rows(gen, count, low, high):
    return torch.randint(low, high, (count,), generator=gen).to(torch.int32)


@pytest.mark.parametrize("dtype,shape", [(torch.float32, (2, 8)), (torch.bfloat16, (8, 128)), (torch.int8, (1, 3)),
                                         (torch.float16, (1, 2)), (torch.bfloat16, (8, 1111))])
@pytest.mark.parametrize("pages,count", [(1, 1), (64, 20), (500, 1500)])
def test_copy(dtype, shape, pages, count):
    caches, *_ = state([], 4, 1, pages, dtype=dtype, shape=shape, tensors=3)
    gen = torch.Generator().manual_seed(1)
    src, dst = random_rows(gen, count, -2, pages + 2), random_rows(gen, count, -2, pages + 2)
    status = both(cf.cache_copy, plain._copy_reference, [caches, src, dst])
    assert count < 20 or 0 in status.tolist()
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    half = pages // 2
    both(cf.cache_copy, plain._copy_reference, [caches, order[:half], order[half : 2 * half]])


@pytest.mark.parametrize("block", [1, 3, 16, 64])
@pytest.mark.parametrize("dtype,shape", [(torch.float32, (2, 8)), (torch.bfloat16, (3, 5)), (torch.uint8, (1, 1))])
def test_fork(block, dtype, shape):
    gen = torch.Generator().manual_seed(block)
    lengths = [int(n) for n in random_rows(gen, 12, 1, 6 * block + 2)] + [0] * 30 + [block, 2 * block, -3]
    caches, counts, tables, context = state(lengths, block, 7, 200, dtype=dtype, shape=shape)
    tables[1, 0] = -1         # names no page
    tables[2, (lengths[2] - 1) // block] = 10**6
    parents, children = random_rows(gen, 60, -1, 46), random_rows(gen, 60, 8, 47)
    both(cf.cache_fork, plain._fork_reference, [caches, counts, tables, context, parents, children])


@pytest.mark.parametrize("free", [0, 1, 5, 17])
def test_fork_until_no_page_is_free(free):
    lengths = [5, 8, 7, 4] + [0] * 40
    caches, counts, tables, context = state(lengths, 4, 3, 7 + free)
    parents = ints(*[i % 4 for i in range(40)])
    children = ints(*[4 + (7 * i) % 40 for i in range(40)])
    both(cf.cache_fork, plain._fork_reference, [caches, counts, tables, context, parents, children])


def test_fork_of_a_row_past_its_table_and_of_many_pairs():
    caches, counts, tables, context = state([5, 12] + [0] * 3000, 4, 3, 4000, shape=(1, 2))
    context[1] = 1000  # past the table
    gen = torch.Generator().manual_seed(0)
    parents, children = random_rows(gen, 5000, 0, 2), random_rows(gen, 5000, 0, 3002)
    both(cf.cache_fork, plain._fork_reference, [caches, counts, tables, context, parents, children])


@pytest.mark.parametrize("tokens", [1, 2, 9, 100])
@pytest.mark.parametrize("block", [1, 4, 16])
def test_extend(tokens, block):
    gen = torch.Generator().manual_seed(tokens)
    lengths = [int(n) for n in random_rows(gen, 40, -2, 6 * block + 1)]
    _, counts, tables, context = state(lengths, block, 6 + 100 // block, 400)
    tables[3] = -1
    for pages in (400, 150):
        sequences = random_rows(gen, 60, -2, 43)
        counts[pages:] = 1
        both(cf.cache_extend, plain._extend_reference, [counts, tables, context, sequences], (block, tokens))


def test_extend_finds_pages_anywhere():
    """Free pages far behind, counts that do not start at a 16-byte boundary."""
    pages = 100_003
    counts = torch.ones(pages + 1, dtype=torch.int32)
    counts[[5, 17000, 99990, 100002]] = 0
    tables, context = torch.zeros(6, 4, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)
    for first in (0, 1):
        arguments = [counts, tables, context, ints(0, 1, 2, 3, 4, 5)]
        gpu, cpu = to("cuda", arguments), to("cpu", arguments)
        gpu[0], cpu[0] = gpu[0][first:], cpu[0][first:]
        same([cf.cache_extend(*gpu, 4, 1)], [plain._extend_reference(*cpu, 4, 1)])
        same(gpu, cpu)


@pytest.mark.parametrize("block", [1, 16])
def test_release(block):
    gen = torch.Generator().manual_seed(0)
    lengths = [int(n) for n in random_rows(gen, 50, -1, 300)]
    _, counts, tables, context = state(lengths, block, 300, 20000)
    tables[4, :2] = torch.tensor([-1, 10**6])
    counts += torch.randint(-1, 3, counts.shape, generator=gen).to(torch.int32)
    tables[5] = tables[6]  # rows that share their pages
    tables[7] = tables[6]
    context[3] = 10**6     # past the table
    sequences = random_rows(gen, 70, -2, 52)
    both(cf.cache_release, plain._release_reference, [counts, tables, context, sequences], (block,))


@pytest.mark.parametrize("pages", [1, 20, 4096, 4097, 30000])
@pytest.mark.parametrize("share", [0.0, 0.3, 0.95, 1.0])
def test_compact(pages, share):
    gen = torch.Generator().manual_seed(pages)
    counts = torch.where(torch.rand(pages, generator=gen) < share, torch.randint(1, 5, (pages,), generator=gen),
                         torch.randint(-2, 1, (pages,), generator=gen)).to(torch.int32)
    caches, _, _, _ = state([], 2, 1, pages, shape=(1, 4), dtype=torch.float16)
    tables = torch.randint(-3, pages + 3, (17, 30), generator=gen).to(torch.int32)
    context = random_rows(gen, 17, -2, 70)
    both(cf.cache_compact, plain._compact_reference, [caches, counts, tables, context])


def test_compact_in_place_and_empty_tables():
    from cuda_force_amd import _lib
    from tests.gpu_util import call, stream

    caches, counts, tables, context = state([30, 7, 0, 50], 4, 13, 9000, shape=(2, 8))
    ref = plain._compact_reference(*to("cpu", [caches, counts, tables, context]))
    gpu = to("cuda", [caches, counts, tables, context])
    live = torch.empty(1, dtype=torch.int32, device="cuda")
    size = _lib.load().cf_cache_workspace_bytes(9000, 4, 0)
    ws = torch.full((size,), 0xA5, dtype=torch.uint8, device="cuda")
    call("cf_cache_compact", _lib.pointer_array([c.data_ptr() for c in gpu[0]]), 2, gpu[0][0][0].nbytes,
         gpu[1].data_ptr(), gpu[2].data_ptr(), gpu[3].data_ptr(), 9000, 4, 4, 13, gpu[1].data_ptr(), gpu[2].data_ptr(),
         live.data_ptr(), ws.data_ptr(), size, stream())
    same([gpu[1], gpu[2], live], ref)
    none = cf.cache_compact(gpu[0], gpu[1], gpu[2][:0], gpu[3][:0])
    assert none[1].shape == (0, 13) and torch.equal(none[2], live)


def test_more_caches_than_a_launch_takes():
    arguments = [*state([9, 0, 0], 4, 4, 12, tensors=70, shape=(1, 4))]
    both(cf.cache_fork, plain._fork_reference, [*arguments, ints(0, 0), ints(1, 2)])
    both(cf.cache_copy, plain._copy_reference, [arguments[0], ints(0, 1, 2), ints(3, 4, 5)])
    both(cf.cache_compact, plain._compact_reference, arguments)


def test_pages_behind_4_gib():
    page = 1 << 20
    cache = torch.zeros(4200, page, dtype=torch.uint8, device="cuda")
    cache[4190], cache[3] = 7, 9
    status = cf.cache_copy([cache], ints(4190, 3).cuda(), ints(5, 4199).cuda())
    assert status.tolist() == [0, 0]
    assert (cache[5] == 7).all() and (cache[4199] == 9).all() and (cache[4198] == 0).all()


def test_general_way_and_saved_tensors():
    caches, counts, tables, context = to("cuda", [*state([9, 0, 0], 4, 4, 12)])
    wide = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    wide[:, 0] = ints(1, 2)
    versions = [t._version for t in (caches[0], counts, tables, context)]
    status = cf.cache_fork(caches, counts, tables, context, ints(0, 0).cuda(), wide[:, 0])
    assert status.tolist() == [0, 0] and context.tolist() == [9, 9, 9]
    assert all(t._version > v for t, v in zip((caches[0], counts, tables, context), versions))


def test_another_stream_and_a_replayed_graph():
    start = state([30, 17, 0, 0, 0, 0], 4, 12, 60)
    caches, counts, tables, context = to("cuda", [*start])
    parents, children = ints(0, 1, 0).cuda(), ints(2, 3, 5).cuda()

    def step():
        status = cf.cache_fork(caches, counts, tables, context, parents, children)
        slots = cf.cache_extend(counts, tables, context, children, 4, 3)
        new = cf.cache_compact(caches, counts, tables, context)
        cf.cache_release(counts, tables, context, children[:1], 4)
        return [status, slots, *new]

    def reset(gpu):
        for t, s in zip([*gpu[0], *gpu[1:]], [*start[0], *start[1:]]):
            t.copy_(s)

    state_ = [caches, counts, tables, context]
    eager = [t.clone() for t in step()]
    after = to("cuda", state_)
    reset(state_)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    same(other, eager)
    reset(state_)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        reset(state_)
        graph.replay()
        torch.cuda.synchronize()
        same(out, eager)
        same(state_, after)


@pytest.mark.parametrize("count", [1023, 1024, 1025, 4000])
@pytest.mark.parametrize("rows", [8192, 8193])
def test_lists_and_tables_on_both_sides_of_what_a_plan_keeps_to_itself(count, rows):
    """Plans of up to 1024 pages over up to 8192 rows (or a copy's pages) work
    in LDS, longer ones in memory."""
    gen = torch.Generator().manual_seed(count)
    lengths = [int(n) for n in random_rows(gen, 300, 1, 12)] + [0] * (rows - 300)
    caches, counts, tables, context = state(lengths, 4, 3, rows, shape=(1, 2))
    parents = random_rows(gen, count, 0, 301)
    children = random_rows(gen, count, 299, rows + 1)
    children[:20] = rows - 1  # the same row again and again, the last one
    both(cf.cache_fork, plain._fork_reference, [caches, counts, tables, context, parents, children])
    sequences = random_rows(gen, count, -1, rows + 1)
    sequences[5:9] = rows - 1
    for tokens in (1, 4, 5):
        both(cf.cache_extend, plain._extend_reference, [counts, tables, context, sequences], (4, tokens))
    src, dst = random_rows(gen, count, 0, rows), random_rows(gen, count, 0, rows)
    dst[3] = src[7] = rows - 1
    both(cf.cache_copy, plain._copy_reference, [caches, src, dst])


def test_lists_that_take_more_than_one_launch():
    """More workgroups (an entry takes one for each of 64 tensors) than a launch
    may have: 2^24 of 256 threads."""
    n = 2**18 + 5
    caches = [torch.zeros(2 * n, 2, 1, 1, device="cuda") for _ in range(64)]
    for i, cache in enumerate(caches):
        cache.copy_(torch.arange(2 * n, device="cuda").view(-1, 1, 1, 1) + i)
    src = torch.arange(n, dtype=torch.int32, device="cuda")
    assert (cf.cache_copy(caches, src, src + n) == 0).all()
    for i, cache in enumerate(caches):
        assert torch.equal(cache[n:], cache[:n]) and cache[n - 1, 0, 0, 0] == n - 1 + i
    # One token in a page of two: every child gets a page of its own.
    counts = torch.zeros(2 * n, dtype=torch.int32, device="cuda")
    counts[0] = 1
    tables = torch.zeros(n + 1, 1, dtype=torch.int32, device="cuda")
    context = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    context[0] = 1
    for i, cache in enumerate(caches):
        cache[0] = -1.0 - i
    assert (cf.cache_fork(caches, counts, tables, context, torch.zeros_like(src), src + 1) == 0).all()
    assert torch.equal(tables[1:, 0], src + 1) and (context == 1).all()
    for i, cache in enumerate(caches):
        assert (cache[: n + 1, 0] == -1.0 - i).all() and (cache[n + 1 :, 0] >= 0).all()
    sequences = torch.full((2**24 + 10,), -1, dtype=torch.int32, device="cuda")
    sequences[3], sequences[-1] = 7, n
    cf.cache_release(counts, tables, context, sequences, 2)
    assert context.sum() == n - 1 and context[7] == 0 and context[n] == 0
    assert counts.sum() == n - 1 and counts[7] == 0 and counts[n] == 0


@pytest.mark.parametrize("pages", [10, 9000])
def test_a_copy_out_of_range_blocks_no_other(pages):
    caches, *_ = state([], 4, 1, pages, shape=(1, 2))
    arguments = [caches, ints(-1, 2, 3, 6, pages, 4), ints(5, 5, 5, 7, 6, 8)]
    assert both(cf.cache_copy, plain._copy_reference, arguments).tolist() == [1, 0, 1, 1, 1, 0]
