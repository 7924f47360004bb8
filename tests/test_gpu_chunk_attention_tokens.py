"""Attention over a paged cache where there are no more new tokens than
sequences (single tokens, or a few sequences with several), which small row
tiles take, against float64."""

from __future__ import annotations

import pytest
import torch

import cuda_force_amd as cf
from tests.chunk_util import CODES, build, check

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HELD = [None, *CODES]
# 12 rows with one before and one behind them, of 13 sequences.
FEW = [(1, 130), (1, 1), (0, 50), (1, 33), (0, 0), (1, 75), (1, 31), (1, 32), (1, 257), (3, 40), (0, 5), (0, 9), (0, 1)]


def run(c):
    assert c.query.shape[0] <= c.context.shape[0]
    got = cf.paged_attention_chunk(*c.args())
    again = cf.paged_attention_chunk(*c.args())
    assert torch.equal(got, again)
    check(got, c)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("dim", [64, 128, 256, 32, 96, 80, 16, 8, 112, 176, 200, 20, 320])
def test_head_sizes(dtype, held, dim):
    run(build(FEW, 4, 2, dim, 16, dtype, held, before=1, behind=1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (12, 4), (16, 1), (17, 1), (32, 1), (60, 2), (33, 1), (70, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_head_layouts(dtype, held, heads, kv_heads, dim):
    run(build([(1, 60), (2, 129), (0, 0), (1, 300), (0, 7)], heads, kv_heads, dim, 16, dtype, held))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("block", [1, 3, 7, 16, 100, 1024])
def test_block_sizes(dtype, held, block):
    run(build([*FEW, (1, 1500)], 8, 2, 64, block, dtype, held))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
def test_contexts_of_every_kind(dtype, held):
    lengths = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1000, 1025]
    run(build([(1, n) for n in lengths], 4, 1, 128, 16, dtype, held))
    run(build([(1, n) for n in lengths] * 4, 6, 2, 64, 16, dtype, held))
    # Few of them, which are cut into ranges.
    for n in (255, 257, 1023, 5000, 20001):
        run(build([(1, n)], 8, 2, 128, 16, dtype, held))
    run(build([(1, 3000 + 700 * i) for i in range(4)], 4, 4, 256, 32, dtype, held))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
def test_several_tokens_of_a_few_sequences(dtype, held):
    for n in (2, 5, 40, 150):
        idle = [(0, 3)] * n
        run(build([(n, n + 100), *idle], 4, 1, 64, 16, dtype, held))
        run(build([*idle, (n, n), (0, 2)], 24, 1, 128, 16, dtype, held))
        run(build([(n, n // 2), *idle], 4, 2, 64, 16, dtype, held))  # more rows than context


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("dim", [64, 128, 256, 80])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_stays_out(dtype, held, dim, bad):
    for new, before, heads in ((3, 30, 4), (10, 30, 4), (6, 60, 24)):
        c = build([(new, new + before), *[(0, 4)] * new], heads, 1, dim, 16, dtype, held)
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
        # In values alone, of one head dimension.
        if held is None:
            c.k[page, at] = 0.0
            c.v[page, at] = 0.0
            zero = cf.paged_attention_chunk(*c.args()).cpu()
            c.v[page, at, :, dim - 1] = bad
            got = cf.paged_attention_chunk(*c.args()).cpu()
            assert torch.equal(got[:row], zero[:row])
            assert not torch.isfinite(got[row:, :, dim - 1]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("held", HELD)
def test_as_stored_wrongly(dtype, held):
    c = build([(4, 100), (6, 120), (3, 80), *[(0, 1)] * 10], 4, 2, 64, 16, dtype, held, bad=False)
    c.tables[1, 2] = 10**6
    c.tables[0, 1] = -1
    c.tables[2, 4] = c.k.shape[0]
    run(c)
    c.context[2] = 2**31 - 1
    c.context[0] = -5
    run(c)
    for starts in ([5, 2, 9, 1], [-3, 4, 4, 2**31 - 1], [13, 13, 13, 13], [-(2**31), 7, 3, 100]):
        c.starts[:4] = torch.tensor(starts, dtype=torch.int32)
        run(c)
    c.tables[:] = -1
    assert (cf.paged_attention_chunk(*c.args()) == 0).all()


@pytest.mark.parametrize("held", HELD)
def test_scores_far_apart_and_queries_of_any_size(held):
    sequences = [(1, 120), (2, 130), (0, 1)]
    for dtype in DTYPES:
        c = build(sequences, 4, 2, 64, 16, dtype, held)
        for scale in (-c.scale, 0.0):
            c.scale = scale
            run(c)
        for size in (300.0, 1e-4, 1e4, 1e30, 1e-37, 0.0):
            if dtype == torch.float16 and size not in (300.0, 1e-4, 0.0):
                continue
            c = build(sequences, 4, 2, 64, 16, dtype, held)
            c.query = (c.query.float() * size).to(dtype)
            c.scale = 0.125 / size if size else 1.0
            run(c)


@pytest.mark.parametrize("held", CODES)
@pytest.mark.parametrize("new", [1, 40])
def test_a_cache_past_64_gigabytes(held, new):
    """Its rows' places pass 2^32 times 16 bytes: K and V are one tensor here."""
    block, heads, dim = 64, 1, 256
    pages = (65 << 30) // (block * heads * dim)
    small = build([(new, 300), (1, 100)], 8, heads, dim, block, torch.bfloat16, held, bad=False)
    small.v, small.v_scales = small.k, small.k_scales
    k = torch.empty(pages, block, heads, dim, dtype=torch.uint8, device="cuda").view(held)
    s = torch.empty(pages, block, heads, device="cuda")
    few = small.k.shape[0]
    at = torch.cat([torch.arange(few // 2), pages - few + torch.arange(few // 2, few)])
    for p, to in enumerate(at.tolist()):
        k.view(torch.uint8)[to].copy_(small.k.view(torch.uint8)[p])
        s[to].copy_(small.k_scales[p])
    there = (small.tables >= 0) & (small.tables < few)
    tables = torch.where(there, at[small.tables.long().clamp(0, few - 1)], -1).to(torch.int32)
    got = cf.paged_attention_chunk(small.query.cuda(), k, k, small.starts.cuda(), tables.cuda(), small.context.cuda(),
                                   s, s, small.scale)
    check(got, small)
    del k, s
    torch.cuda.empty_cache()
