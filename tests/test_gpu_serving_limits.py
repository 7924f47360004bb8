"""Operators of serving in 8 bits at sizes past 32 bits and past one launch."""

from __future__ import annotations

import pytest
import torch

import cuda_force_amd as cf
from tests.chunk_util import CODES, build, check

pytestmark = pytest.mark.gpu


def ints(m, k):
    return torch.randint(-128, 128, (m, k), device="cuda", dtype=torch.int8)


def test_products_of_any_depth_past_one_launch():
    """Results in tiles of 16 x 16: more of them than one launch has workgroups."""
    m, n, k = 70000, 40000, 17
    x, w = ints(m, k), ints(n, k)
    ones = torch.ones(m, device="cuda")
    y = cf.matmul_int8(x, w, ones, ones[:n])
    for at in (0, 15, 53687, 53688, 67000, m - 1):
        want = (x[at].double() @ w.double().t()).to(torch.bfloat16)
        assert torch.equal(y[at], want)
    del y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("k", [16, 3])
def test_one_row_by_columns_past_one_launch(k):
    n = 2**27 + 2**26 + 5
    x, w = ints(1, k), ints(n, k)
    ones = torch.ones(n, device="cuda")
    y = cf.matmul_int8(x, w, ones[:1], ones, dtype=torch.float32)
    for a in range(0, n, 2**25):
        assert torch.equal(y[0, a : a + 2**25], (w[a : a + 2**25].float() * x.float()).sum(1))
    del y, w, ones
    torch.cuda.empty_cache()


def test_more_wide_rows_than_a_launch_of_large_workgroups_has():
    """Rows of more than 8192 fp32 numbers have a workgroup of 1024 threads each."""
    rows, cols = 2**22 + 3, 8200
    if torch.cuda.mem_get_info()[0] < 190 << 30:
        pytest.skip("needs 190 GiB of memory")
    x = torch.empty(rows, cols, device="cuda")
    at = [0, 1, 2**21, 2**22 - 2, 2**22 - 1, 2**22, rows - 1]
    x[at] = torch.randn(len(at), cols, device="cuda")
    codes, scales = cf.quantize_int8_rows(x)
    want, want_scales = cf.quantize_int8_rows(x[at].cpu())
    assert torch.equal(codes[at].cpu(), want) and torch.equal(scales[at].cpu(), want_scales)
    del x, codes
    torch.cuda.empty_cache()


@pytest.mark.parametrize("held", [torch.bfloat16, *CODES])
@pytest.mark.parametrize("new", [1, 40])
def test_rows_past_4_gigabytes_of_a_cache(held, new):
    """Written, read back and attended to: at the cache's beginning, over byte 2^32
    (within a row) and in the last pages, as in a small cache."""
    block, heads, dim = 64, 8, 96
    pages = 87400
    token = heads * dim * held.itemsize
    assert pages * block * token > 2**32 and 2**32 % token != 0
    k, v = (torch.zeros(pages, block, heads, dim, dtype=torch.uint8, device="cuda").view(held) if held in CODES else
            torch.zeros(pages, block, heads, dim, dtype=held, device="cuda") for _ in range(2))
    scales = [torch.ones(pages, block, heads, device="cuda") if held in CODES else None for _ in range(2)]
    over = 2**32 // token // block
    at = torch.tensor([0, over - 1, over, over + 1, pages - 2, pages - 1])
    small = [torch.zeros(len(at), block, heads, dim, device="cuda").to(held) for _ in range(2)]
    small += [None if s is None else torch.ones(len(at), block, heads, device="cuda") for s in scales]
    n = len(at) * block
    x = torch.randn(n, 2, heads, dim, device="cuda", dtype=torch.bfloat16)
    places = torch.arange(n, device="cuda")
    slots = at.cuda()[places // block] * block + places % block
    cf.cache_write(x[:, 0], x[:, 1], k, v, slots, *scales)
    cf.cache_write(x[:, 0], x[:, 1], small[0], small[1], places, *small[2:])
    for big, few in zip((k, v, *scales), small):
        if big is not None:
            raw = big if held == torch.bfloat16 or big.dtype == torch.float32 else big.view(torch.uint8)
            assert torch.equal(raw[at.cuda()], few.view(raw.dtype))
    got = cf.cache_read(k, v, slots, *scales, dtype=torch.bfloat16)
    want = cf.cache_read(small[0], small[1], places, *small[2:], dtype=torch.bfloat16)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0].abs().sum() > 0
    q = torch.randn(new, 32, dim, device="cuda", dtype=torch.bfloat16)
    starts, context = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, new], [n]))
    tables = torch.arange(len(at), dtype=torch.int32, device="cuda")[None]
    got = cf.paged_attention_chunk(q, k, v, starts, at.to(torch.int32).cuda()[None], context, *scales)
    assert torch.equal(got, cf.paged_attention_chunk(q, small[0], small[1], starts, tables, context, *small[2:]))
    del k, v, scales
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("held", [None, *CODES])
@pytest.mark.parametrize("sequences", [[(1, 5000)], [(3, 700), (1, 3000), (0, 9)], [(40, 900)], [(5, 6), (1, 1)]])
def test_misaligned_query_and_caches(dtype, held, sequences):
    """An element behind a whole vector: the general kernel, in as many ranges as
    the matrix kernels' plan has."""
    c = build(sequences, 8, 2, 64, 16, dtype, held)
    for which in ([0], [1], [2], [0, 1, 2]):
        args = c.args()
        for i in which:
            flat = torch.zeros(args[i].numel() + 1, device="cuda").to(args[i].dtype)
            args[i] = flat[1:].view(args[i].shape).copy_(args[i])
            assert args[i].data_ptr() % 16 != 0
        got = cf.paged_attention_chunk(*args)
        check(got, c)
        assert torch.equal(got, cf.paged_attention_chunk(*args))
