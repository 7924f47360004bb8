"""Pages of a paged cache on the CPU: what each operator does, and refusals."""

from __future__ import annotations

import ctypes

import pytest
import torch

import cuda_force_amd as cf
from cuda_force_amd import _lib
from tests.pages_util import ints, state, to


def test_copy():
    caches, *_ = state([], 4, 1, 10)
    before = [c.clone() for c in caches]
    #      good, dst taken, src is a dst, out of range (4), onto itself, good
    src = ints(0, 1, 5, -1, 10, 2, 2, 7, 0)
    dst = ints(5, 5, 6, 3, 3, 10, -2, 7, 9)
    status = cf.cache_copy(caches, src, dst)
    assert status.tolist() == [0, 1, 1, 1, 1, 1, 1, 1, 0]
    for cache, old in zip(caches, before):
        expect = old.clone()
        expect[5], expect[9] = old[0], old[0]
        assert torch.equal(cache, expect)


def test_fork_shares_whole_pages_and_copies_the_partial_one():
    caches, counts, tables, context = state([10, 8, 0, 0, 0], 4, 5, 12)
    old = [c.clone() for c in caches]
    free = [p for p in range(12) if counts[p] == 0]
    rows = tables.clone()
    status = cf.cache_fork(caches, counts, tables, context, ints(0, 1, 0), ints(4, 2, 3))
    assert status.tolist() == [0, 0, 0] and context.tolist() == [10, 8, 8, 10, 10]
    assert tables[4, :2].tolist() == tables[3, :2].tolist() == rows[0, :2].tolist()
    assert tables[2, :2].tolist() == rows[1, :2].tolist()
    assert tables[4, 2] == free[0] and tables[3, 2] == free[1]
    assert [int(counts[p]) for p in rows[0, :3]] == [3, 3, 1] and [int(counts[p]) for p in rows[1, :2]] == [2, 2]
    assert counts[free[0]] == counts[free[1]] == 1 and counts.sum() == 3 * 2 + 1 + 2 * 2 + 2
    for cache, was in zip(caches, old):
        for page in free[:2]:
            assert torch.equal(cache[page, :2], was[rows[0, 2], :2]) and torch.equal(cache[page, 2:], was[page, 2:])
            was[page] = cache[page]
        assert torch.equal(cache, was)


def test_fork_leaves_out_what_it_cannot_do():
    caches, counts, tables, context = state([5, 4, 0, 0, 0, 0], 4, 3, 4)  # one page free
    parents = ints(0, 2, 1, 0, 0, -1, 0, 6, 1, 0)
    children = ints(2, 3, 0, 2, 3, 4, 6, 4, 4, 5)
    # done; empty parent; child in use; child taken; no page; ranges (3); done; no page
    status = cf.cache_fork(caches, counts, tables, context, parents, children)
    assert status.tolist() == [0, 1, 1, 1, 2, 1, 1, 1, 0, 2]
    assert context.tolist() == [5, 4, 5, 0, 4, 0]


def test_extend():
    caches, counts, tables, context = state([3, 4, 0, 20], 4, 5, 9)  # one page free, row 3 full
    page = int(tables[0, 0])
    free = [p for p in range(9) if counts[p] == 0]
    slots = cf.cache_extend(counts, tables, context, ints(0, 3, 1, 7, 0, 2, -1), 4)
    assert len(free) == 2
    assert slots.view(-1).tolist() == [page * 4 + 3, -1, free[0] * 4, -1, -1, free[1] * 4, -1]
    assert context.tolist() == [4, 5, 1, 20] and (counts > 0).all()
    assert cf.cache_extend(counts, tables, context, ints(0, 1), 4).view(-1).tolist() == [-1, free[0] * 4 + 1]


def test_extend_by_many_tokens_is_all_or_nothing():
    caches, counts, tables, context = state([0, 2, 0], 4, 6, 7)  # six pages free
    slots = cf.cache_extend(counts, tables, context, ints(1, 0, 2), 4, 11)
    free = [p for p in range(7) if p != int(tables[1, 0])]
    assert context.tolist() == [11, 13, 0] and (slots[2] == -1).all()
    pages = [int(tables[1, 0])] + free[:3]
    assert slots[0].tolist() == [pages[t // 4] * 4 + t % 4 for t in range(2, 13)]
    assert slots[1].tolist() == [free[3 + t // 4] * 4 + t % 4 for t in range(11)]


def test_release_and_reuse():
    caches, counts, tables, context = state([9, 5, 0], 4, 4, 8)
    cf.cache_fork(caches, counts, tables, context, ints(0), ints(2))
    rows = tables.clone()
    cf.cache_release(counts, tables, context, ints(0, 0, 5, -1), 4)
    assert context.tolist() == [0, 5, 9] and torch.equal(tables, rows)
    assert [int(counts[p]) for p in rows[0, :3]] == [1, 1, 0]
    cf.cache_release(counts, tables, context, ints(2, 1), 4)
    assert (counts == 0).all() and (context == 0).all()
    cf.cache_release(counts, tables, context, ints(0, 1, 2), 4)
    assert (counts == 0).all()


def test_compact():
    caches, counts, tables, context = state([9, 5, 0, 12], 4, 4, 20)
    cf.cache_fork(caches, counts, tables, context, ints(0), ints(2))
    before = to("cpu", [caches, counts, tables, context])
    new_counts, new_tables, live = cf.cache_compact(caches, counts, tables, context)
    assert live.tolist() == [9] and (new_counts[:9] > 0).all() and (new_counts[9:] == 0).all()
    assert torch.equal(counts, before[1]) and torch.equal(tables, before[2])
    for s, n in enumerate(context.tolist()):
        held = -(-n // 4)
        assert (new_tables[s, :held] < 9).all() and torch.equal(new_tables[s, held:], tables[s, held:])
        for cache, was in zip(caches, before[0]):
            assert torch.equal(cache[new_tables[s, :held].long()], was[tables[s, :held].long()])
        assert torch.equal(new_counts[new_tables[s, :held].long()], counts[tables[s, :held].long()])


def test_empty_lists():
    caches, counts, tables, context = state([3], 4, 2, 3)
    none = ints()
    assert cf.cache_copy(caches, none, none).shape == (0,)
    assert cf.cache_fork(caches, counts, tables, context, none, none).shape == (0,)
    assert cf.cache_extend(counts, tables, context, none, 4, 3).shape == (0, 3)
    cf.cache_release(counts, tables, context, none, 4)
    assert context.tolist() == [3]


def test_refusals():
    caches, counts, tables, context = state([3, 0], 4, 2, 3)
    one, two = ints(0), ints(0, 1)
    for bad in ([], caches[0], [caches[0], caches[1][:2]], [caches[0], caches[1].double()],
                [c.transpose(0, 1) for c in caches], [c.clone().requires_grad_(True) for c in caches]):
        with pytest.raises(ValueError):
            cf.cache_copy(bad, one, one)
        with pytest.raises(ValueError):
            cf.cache_fork(bad, counts, tables, context, one, one)
        with pytest.raises(ValueError):
            cf.cache_compact(bad, counts, tables, context)
    for call in (lambda: cf.cache_copy(caches, one, two), lambda: cf.cache_copy(caches, one[None], one[None]),
                 lambda: cf.cache_fork(caches, counts[:2], tables, context, one, one),
                 lambda: cf.cache_fork(caches, counts, tables[:1], context, one, one),
                 lambda: cf.cache_fork(caches, counts, tables, context, one, two),
                 lambda: cf.cache_fork(caches, counts, tables.t(), context, one, one),
                 lambda: cf.cache_fork([c[:, 0, 0, 0].contiguous() for c in caches], counts, tables, context, one, one),
                 lambda: cf.cache_extend(counts, tables, context, one, 0),
                 lambda: cf.cache_extend(counts, tables, context, one, 4, 0),
                 lambda: cf.cache_extend(counts, tables, context[:1], one, 4),
                 lambda: cf.cache_release(counts, tables, context, one, -1),
                 lambda: cf.cache_compact(caches, counts[:1], tables, context)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: cf.cache_copy(caches, one.long(), one), lambda: cf.cache_fork(
            caches, counts.long(), tables, context, one, one), lambda: cf.cache_extend(
            counts, tables.long(), context, one, 4), lambda: cf.cache_release(
            counts, tables, context, one.long(), 4), lambda: cf.cache_compact(caches, counts, tables, context.long())):
        with pytest.raises(TypeError):
            call()


def test_c_abi_refusals_before_any_launch():
    lib = _lib.load()
    p, null = ctypes.c_void_p(0x1000), ctypes.c_void_p(0)
    bad = _lib.CF_ERR_INVALID_ARGUMENT
    caches = _lib.pointer_array([0x1000, 0x2000])

    def copy(caches=caches, n=2, page=1024, pages=10, src=p, count=3, status=p, ws=p, size=1 << 20):
        return lib.cf_cache_copy(caches, n, page, pages, src, p, count, status, ws, size, null)

    assert copy(count=0) == _lib.CF_OK
    for case in ({"caches": None}, {"n": -1}, {"page": 0}, {"pages": 0}, {"pages": 2**30 + 1}, {"src": null},
                 {"status": null}, {"ws": null}, {"size": 16}, {"ws": ctypes.c_void_p(0x1008)}, {"count": 2**30 + 1},
                 {"caches": _lib.pointer_array([0x1000, 0])}):
        assert copy(**case) == bad, case

    def fork(counts=p, tables=p, block=4, pages=10, rows=3, width=5, page=1024, parents=p, count=2, size=1 << 20):
        return lib.cf_cache_fork(caches, 2, page, counts, tables, p, pages, block, rows, width, parents, p, count, p,
                                 p, size, null)

    assert fork(count=0) == _lib.CF_OK
    for case in ({"counts": null}, {"tables": null}, {"block": 0}, {"pages": 0}, {"rows": 0}, {"width": 0},
                 {"page": 1023}, {"parents": null}, {"size": 0}, {"count": 2**31}):
        assert fork(**case) == bad, case

    def extend(block=4, tokens=1, slots=p, count=2, size=1 << 20, rows=3):
        return lib.cf_cache_extend(p, p, p, 10, block, rows, 5, p, count, tokens, slots, p, size, null)

    assert extend(count=0) == _lib.CF_OK
    for case in ({"block": 0}, {"tokens": 0}, {"slots": null}, {"size": 0}, {"tokens": 2**30}, {"rows": 0}):
        assert extend(**case) == bad, case
    assert lib.cf_cache_release(p, p, p, 10, 4, 3, 5, p, 0, null) == _lib.CF_OK
    assert lib.cf_cache_release(p, p, p, 10, 0, 3, 5, p, 1, null) == bad
    assert lib.cf_cache_release(p, p, p, 10, 4, 3, 5, null, 1, null) == bad

    def compact(counts=p, new=p, live=p, pages=10, tables=p, size=1 << 20):
        return lib.cf_cache_compact(caches, 2, 1024, counts, tables, p, pages, 4, 3, 5, new, p, live, p, size, null)

    for case in ({"counts": null}, {"new": null}, {"live": null}, {"pages": 0}, {"tables": null}, {"size": 0}):
        assert compact(**case) == bad, case


def test_a_copy_out_of_range_blocks_no_other():
    caches, *_ = state([], 4, 1, 10)
    before = [c.clone() for c in caches]
    #      out of range, good all the same, taken, from a page that one names as its dst, out of range
    src, dst = ints(-1, 2, 3, 6, 10, 4), ints(5, 5, 5, 7, 6, 8)
    assert cf.cache_copy(caches, src, dst).tolist() == [1, 0, 1, 1, 1, 0]
    for cache, old in zip(caches, before):
        expect = old.clone()
        expect[5], expect[8] = old[2], old[4]
        assert torch.equal(cache, expect)
