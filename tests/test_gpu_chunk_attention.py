"""Attention of chunks of new tokens on the GPU against float64."""

from __future__ import annotations

import pytest
import torch

import cuda_force_amd as cf
from tests.chunk_util import CODES, build, check

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HELD = [None, *CODES]
MIXED = [(40, 100), (1, 130), (0, 50), (33, 33), (1, 1), (70, 75), (2, 61)]


def run(c):
    got = cf.paged_attention_chunk(*c.args())
    again = cf.paged_attention_chunk(*c.args())
    assert torch.equal(got, again)
    check(got, c)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("dim", [64, 128, 256, 32, 96, 80, 8, 20, 130, 512])
def test_head_sizes(dtype, held, dim):
    run(build(MIXED, 4, 2, dim, 16, dtype, held, before=3, behind=5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (12, 4), (16, 2), (17, 1), (40, 1), (70, 2)])
def test_head_layouts(dtype, held, heads, kv_heads):
    run(build([(5, 60), (1, 129), (17, 20)], heads, kv_heads, 64, 16, dtype, held))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("block", [1, 2, 3, 7, 16, 24, 64, 100, 1024])
def test_block_sizes(dtype, held, block):
    run(build([(40, 140), (1, 71), (33, 70)], 4, 2, 64, block, dtype, held, behind=1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
def test_chunk_and_context_lengths(dtype, held):
    for new in (1, 2, 7, 8, 9, 31, 32, 33, 64, 65, 100):
        for before in (0, 1, 31, 32, 33, 95, 200):
            run(build([(new, new + before), (1, before + 1)], 4, 1, 64, 16, dtype, held, seed=new))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
def test_long_contexts_and_many_sequences(dtype, held):
    run(build([(1, 5000 + 7 * i) for i in range(3)] + [(150, 4000)], 8, 2, 128, 16, dtype, held))
    run(build([(i % 4, 3 + 5 * (i % 30)) for i in range(200)], 4, 2, 64, 16, dtype, held))
    run(build([(1, 20000)], 4, 4, 128, 32, dtype, held))
    run(build([(700, 900)], 4, 1, 128, 16, dtype, held))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
def test_more_rows_than_context_and_nothing_to_see(dtype, held):
    got = run(build([(50, 20), (3, 0), (1, 0), (40, 1)], 4, 2, 64, 16, dtype, held))
    assert (got[:30] == 0).all() and (got[50:54] == 0).all()
    c = build([(50, 60), (1, 9)], 4, 2, 64, 16, dtype, held)
    c.tables[:] = -1
    assert (cf.paged_attention_chunk(*c.args()) == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("dim", [64, 20])
def test_starts_tables_and_lengths_as_stored_wrongly(dtype, held, dim):
    c = build([(40, 100), (60, 120), (30, 80)], 4, 2, dim, 16, dtype, held, bad=False)
    c.tables[1, 2] = 10**6
    c.tables[0, 1] = -1
    c.tables[2, 4] = c.k.shape[0]
    run(c)
    c.context[2] = 2**31 - 1
    c.context[0] = -5
    run(c)
    for starts in ([5, 2, 9, 1], [-3, 4, 4, 2**31 - 1], [130, 130, 130, 130], [-(2**31), 7, 3, 100]):
        c.starts = torch.tensor(starts, dtype=torch.int32)
        run(c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_stays_out(dtype, held, bad):
    for new, before in ((40, 100), (6, 30), (150, 0)):
        c = build([(new, new + before)], 4, 2, 64, 16, dtype, held)
        clean = cf.paged_attention_chunk(*c.args()).cpu()
        row = new // 2
        page, at = int(c.tables[0, (before + row) // 16]), (before + row) % 16
        if held is None:
            c.k[page, at], c.v[page, at] = bad, bad
        else:
            c.k_scales[page, at], c.v_scales[page, at] = bad, bad
            if held == torch.float8_e4m3fn:
                c.v.view(torch.uint8)[page, at] = 0x7F
        got = cf.paged_attention_chunk(*c.args()).cpu()
        assert torch.equal(got[:row], clean[:row])
        assert not torch.isfinite(got[row:]).all(-1).any()


@pytest.mark.parametrize("held", HELD)
def test_scores_far_apart_and_queries_of_any_size(held):
    for dtype in DTYPES:
        c = build([(20, 120), (1, 130)], 4, 2, 64, 16, dtype, held)
        c.scale = -c.scale
        run(c)
        c.scale = 0.0
        run(c)
        for size in (300.0, 1e-4, 1e4, 1e30, 1e-37, 0.0):
            if dtype == torch.float16 and size not in (300.0, 1e-4, 0.0):
                continue
            c = build([(20, 120), (1, 130)], 4, 2, 64, 16, dtype, held)
            c.query = (c.query.float() * size).to(dtype)
            c.scale = 0.125 / size if size else 1.0
            run(c)


def test_row_tiles_of_a_context_split_and_not():
    for sequences in ([(300, 3000)], [(130, 2500), (1, 2500)], [(1, 3000)] * 3 + [(0, 5)] * 70):
        for held in HELD:
            run(build(sequences, 8, 1, 64, 16, torch.bfloat16, held))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("dim", [64, 128, 256, 96])
def test_tiles_of_64_rows(dtype, held, dim):
    """Taken for all rows where tables are short and tiles of 128 would be cut."""
    run(build([(130, 300), (97, 300), (1, 200), (160, 160), (0, 9), (33, 290)], 32, 8, dim, 16, dtype, held, before=2, behind=9))
    run(build([(150, 400)] * 2, 16, 16, dim, 16, dtype, held))
    # A tile's second half without tokens, rows without any.
    run(build([(90, 90), (60, 20), (160, 161)], 32, 8, dim, 16, dtype, held))


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_a_row_of_such_a_tile_does_not_see(held, bad):
    for dtype in DTYPES:
        c = build([(150, 170)] * 3, 32, 8, 64, 16, dtype, held)
        clean = cf.paged_attention_chunk(*c.args()).cpu()
        for row in (3, 40, 80):  # in either half of a step's tokens
            page, at = int(c.tables[1, (20 + row) // 16]), (20 + row) % 16
            if held is None:
                c.k[page, at], c.v[page, at] = bad, bad
            else:
                c.k_scales[page, at], c.v_scales[page, at] = bad, bad
                if held == torch.float8_e4m3fn:
                    c.v.view(torch.uint8)[page, at] = 0x7F
        got = cf.paged_attention_chunk(*c.args()).cpu()
        assert torch.equal(got[:153], clean[:153]) and torch.equal(got[300:], clean[300:])
        assert not torch.isfinite(got[153:300]).all(-1).any()


def test_views_misaligned_and_other_streams():
    c = build(MIXED, 4, 2, 64, 16, torch.bfloat16)
    want = cf.paged_attention_chunk(*c.args())
    args = c.args()
    flat = torch.empty(args[0].numel() + 1, dtype=torch.bfloat16, device="cuda")
    args[0] = flat[1:].view(c.query.shape).copy_(args[0])
    check(cf.paged_attention_chunk(*args), c)
    wide = torch.zeros(*c.query.shape[:2], 128, dtype=torch.bfloat16, device="cuda")
    wide[..., :64] = c.query.cuda()
    args[0] = wide[..., :64]
    assert torch.equal(cf.paged_attention_chunk(*args), want)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = cf.paged_attention_chunk(*args)
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("held", HELD)
def test_graph(held):
    c = build([(30, 700), (1, 900), (0, 5)], 8, 2, 64, 16, torch.bfloat16, held, bad=False)
    args = c.args()
    cf.paged_attention_chunk(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cf.paged_attention_chunk(*args)
    for lengths in ([700, 900, 5], [650, 1, 5], [30, 800, 0]):
        args[5].copy_(torch.tensor(lengths, dtype=torch.int32))
        args[0].copy_(torch.randn_like(args[0]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, cf.paged_attention_chunk(*args))


def test_a_row_past_four_gigabytes():
    """Places behind 2^32 bytes of a cache."""
    pages, block, heads, dim = 40000, 64, 8, 128
    k = torch.zeros(pages, block, heads, dim, dtype=torch.int8, device="cuda").view(torch.int8)
    v = torch.zeros_like(k)
    ks, vs = (torch.ones(pages, block, heads, device="cuda") for _ in range(2))
    x = torch.randn(100, 2, heads, dim, device="cuda", dtype=torch.bfloat16)
    slots = (pages - 2) * block + torch.arange(100, device="cuda")
    small = [t[-2:].clone() for t in (k, v, ks, vs)]
    cf.cache_write(x[:, 0], x[:, 1], k, v, slots, ks, vs)
    cf.cache_write(x[:, 0], x[:, 1], small[0], small[1], slots - (pages - 2) * block, small[2], small[3])
    for a, b in zip((k, v, ks, vs), small):
        assert torch.equal(a[-2:], b)
    q = torch.randn(100, 32, dim, device="cuda", dtype=torch.bfloat16)
    starts, context = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, 100], [100]))
    tables = torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32, device="cuda")
    got = cf.paged_attention_chunk(q, k, v, starts, tables, context, ks, vs)
    assert torch.equal(got, cf.paged_attention_chunk(q, small[0], small[1], starts, tables - (pages - 2), context,
                                                     small[2], small[3]))
    assert all(torch.equal(a, b) for a, b in zip(cf.cache_read(k, v, slots, ks, vs),
                                                 cf.cache_read(*small[:2], slots - (pages - 2) * block, *small[2:])))
