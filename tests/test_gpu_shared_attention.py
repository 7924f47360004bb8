"""Attention behind shared prompts on the GPU against float64."""

from __future__ import annotations

import pytest
import torch

import cuda_force_amd as cf
from tests.shared_util import build, check, reference

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def run(c):
    got = cf.paged_attention_shared(*c.args())
    again = cf.paged_attention_shared(*c.args())
    assert torch.equal(got, again)
    check(got, c)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256, 32, 96, 80, 8, 20, 130, 512])
def test_head_sizes(dtype, dim):
    run(build([(100, [100, 130, 99, 161]), (33, [70, 33])], 4, 2, dim, 16, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (12, 4), (16, 2), (17, 1), (40, 1), (70, 2)])
def test_head_layouts(dtype, heads, kv_heads):
    run(build([(50, [60] * 3), (129, [129 + i for i in range(11)])], heads, kv_heads, 64, 16, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block", [1, 2, 3, 7, 16, 24, 64, 100, 1024])
def test_block_sizes(dtype, block):
    run(build([(70, [71, 140, 70]), (1, [1, 2])], 4, 2, 64, block, dtype, loners=2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 31, 32, 33, 64, 127, 128, 129, 500, 1000])
@pytest.mark.parametrize("sequences", [1, 5, 40])
def test_prefix_lengths(dtype, prefix, sequences):
    run(build([(prefix, [prefix + (7 * i) % 50 for i in range(sequences)])], 8, 2, 64, 16, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_contexts_and_many_sequences(dtype):
    run(build([(3000, [3000 + 11 * i for i in range(50)]), (1, [2500, 1])], 8, 2, 128, 16, dtype))
    run(build([(20000, [20001, 20700])], 4, 1, 64, 32, dtype))
    run(build([(10, [5000])], 4, 4, 128, 16, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_contexts_shorter_than_the_prefix(dtype):
    # The first sequences hold too little; one of the group is empty.
    run(build([(300, [10, 0, 299, 300, 400, 310]), (200, [5, 6]), (50, [0, 0])], 8, 2, 64, 16, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_groups_loners_and_copies(dtype):
    run(build([(40, []), (64, [64, 70]), (9, []), (31, [40])], 4, 2, 64, 16, dtype, loners=70))
    run(build([(100, [120, 130, 140])], 4, 2, 64, 16, dtype, copies=True))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_groups(dtype):
    run(build([(20 + g % 5, [30 + i for i in range(g % 4)]) for g in range(150)], 4, 2, 64, 16, dtype))


@pytest.mark.parametrize("fill", [float("inf"), float("-inf"), 1e4])
def test_what_lies_behind_a_context_stays_out(fill):
    for dtype in DTYPES:
        run(build([(33, [34, 77, 20]), (5, [0, 12])], 4, 2, 64, 16, dtype, fill=fill))


@pytest.mark.parametrize("dtype", DTYPES)
def test_groups_as_stored_wrongly_share_nothing_they_should_not(dtype):
    """Starts out of order or out of range, prefixes past the context or the
    table, with every sequence's own tokens different: nothing may be shared
    that the normalised groups do not hold."""
    c = build([(0, [40, 50, 60, 70])], 4, 2, 64, 16, dtype)
    for starts, prefix in (([-5, -1, 0], [30, 30]), ([4, 9, 100], [30, 30]), ([3, 1, 4], [0, 64]),
                           ([0, 1, 2], [2**31 - 1, -7]), ([2, 2, 2], [40, 40])):
        c.starts, c.prefix = torch.tensor(starts, dtype=torch.int32), torch.tensor(prefix, dtype=torch.int32)
        run(c)
    c.starts, c.prefix = torch.tensor([0], dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
    run(c)  # no groups


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 20])
def test_entries_that_name_no_page(dtype, dim):
    c = build([(100, [120, 130, 250])], 4, 2, dim, 16, dtype)
    c.tables[:, 2] = -1
    c.tables[1, 7] = 10**6
    c.tables[2, 7:] = c.k.shape[0]
    run(c)
    c.tables[:] = -1
    assert (cf.paged_attention_shared(*c.args()) == 0).all()


@pytest.mark.parametrize("dim", [64, 20])
def test_lengths_past_the_table_and_below_zero(dim):
    c = build([(64, [128, 128, 128])], 4, 2, dim, 16, torch.bfloat16)
    c.context[0] = 2**31 - 1
    c.context[1] = -3
    run(c)


def test_scores_far_apart_and_not_finite():
    c = build([(100, [120, 130])], 4, 2, 64, 16, torch.float32, fill=0.0)
    c.query *= 300.0
    got = cf.paged_attention_shared(*c.args())
    assert torch.isfinite(got).all()
    c.scale = -c.scale
    c.query /= 300.0
    run(c)
    c.scale = 0.0
    run(c)
    c.scale = 0.125
    page, at = int(c.tables[1, 7]), 118 % 16
    c.k[page, at] = float("nan")  # token 118 of sequence 1 alone
    got = cf.paged_attention_shared(*c.args()).cpu()
    assert got[1].isnan().all() and torch.isfinite(got[0]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_misaligned_tensors(dtype):
    c = build([(40, [50, 60])], 4, 2, 64, 16, dtype)
    args = c.args()
    for i in range(3):
        flat = torch.empty(args[i].numel() + 1, dtype=dtype, device="cuda")[1:]
        args[i] = flat.copy_(args[i].reshape(-1)).view(args[i].shape)
    check(cf.paged_attention_shared(*args), c)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes and elements, its last pages in use."""
    dim, block, kv_heads = 128, 16, 8
    small = build([(40, [50, 60])], 8, kv_heads, dim, block, torch.bfloat16)
    pages = 2**32 // (block * kv_heads * dim) + 50
    args = small.args()
    shift = pages - small.k.shape[0]
    for i in (1, 2):
        big = torch.zeros(pages, block, kv_heads, dim, dtype=torch.bfloat16, device="cuda")
        big[shift:] = args[i]
        args[i] = big
    args[5] = torch.where((args[5] >= 0) & (args[5] < small.k.shape[0]), args[5] + shift, args[5])
    check(cf.paged_attention_shared(*args), small)


def test_general_way_equals_direct():
    c = build([(40, [50, 60])], 4, 2, 64, 16, torch.float16)
    args = c.args()
    direct = cf.paged_attention_shared(*args)
    wide = torch.empty(2, 4, 128, dtype=torch.float16, device="cuda")[..., ::2]
    wide.copy_(args[0])
    assert torch.equal(direct, cf.paged_attention_shared(wide, *args[1:]))
    tables = torch.cat([args[5], args[5]], 1)[:, : args[5].shape[1]]
    assert torch.equal(direct, cf.paged_attention_shared(*args[:5], tables, *args[6:]))
    none = cf.paged_attention_shared(args[0][:0], *args[1:3], args[3][:1] * 0, args[4][:0], args[5][:0], args[6][:0])
    assert none.shape == (0, 4, 64)


def test_another_stream_and_a_replayed_graph():
    c = build([(400, [410, 500, 450, 400])], 8, 2, 128, 16, torch.bfloat16)
    args = c.args()
    eager = cf.paged_attention_shared(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = cf.paged_attention_shared(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(eager, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cf.paged_attention_shared(*args)
    for step, (prefix, context) in enumerate([(400, [410, 500, 450, 400]), (16, [20, 0, 33, 400]),
                                              (64, [64, 65, 450, 70])]):
        c.prefix[0], c.context = prefix, torch.tensor(context, dtype=torch.int32)
        args[4].copy_(c.prefix)
        args[6].copy_(c.context)
        c.query = torch.randn_like(c.query)
        args[0].copy_(c.query)
        graph.replay()
        torch.cuda.synchronize()
        check(out, c)
        assert torch.equal(out, cf.paged_attention_shared(*args)), step


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nats", [8.0, 12.0, 14.0, 16.0, 17.5, 18.0, 25.0])
@pytest.mark.parametrize("prefix", [0, 5000])
def test_a_leading_key_without_a_value(dtype, nats, prefix):
    """One key leads all others by so much that these hold little weight, and
    the result is theirs alone."""
    c = build([(prefix, [5000, 4000 + prefix, 5001 + prefix])], 4, 2, 64, 16, dtype, fill=0.0)
    c.query[:] = 0
    c.query[..., :2] = 1.0
    c.k[..., 0] = 0
    c.v[:] = (c.v.float().abs() / 4 + 0.5).to(dtype)  # nothing cancels
    for s in range(3):
        page = int(c.tables[s, 0])
        c.k[page, 0, :, 0], c.k[page, 0, :, 1], c.v[page, 0] = 8 * nats, 0.0, 0.0
    got = cf.paged_attention_shared(*c.args()).cpu().double()
    ref, size = reference(c)
    # As shared_util.check; and fp16 probabilities below 2^-14 of the 2^13 that
    # stand for the largest are off by half of 2^-24, whatever their size.
    half = torch.finfo(dtype).eps / 2
    f32 = 2.0**-16 + 2.0**-24 * float(c.context.max()) / 32
    tolerance = (f32 + (half if dtype != torch.float32 else 0.0)) * size + half * ref.abs()
    if dtype == torch.float16:
        tolerance += 2.0**-25  # the result's own smallest step, halved
        tolerance += 2.0**-38 * c.context.double()[:, None, None] * c.v.double().abs().max()
    worst = ((got - ref).abs() - tolerance).max().item()
    assert worst <= 0, worst


@pytest.mark.parametrize("grouped", [False, True])
def test_lengths_at_the_end_of_32_bits(grouped):
    """Contexts of 2^31 - 4096 tokens, the most there are, of which the table
    names the first and the last block alone."""
    most, block, dim = 2**31 - 4096, 1 << 16, 64
    gen = torch.Generator().manual_seed(0)
    query = torch.randn(3, 2, dim, generator=gen).bfloat16()
    k, v = (torch.randn(2, block, 1, dim, generator=gen).bfloat16() for _ in range(2))
    tables = torch.full((3, 1 << 15), -1, dtype=torch.int32)
    tables[:, 0], tables[:, -1] = 1, 0
    lengths = [most, 2**31 - 1, 70000]
    starts, prefix = ([0, 3], [most - 1]) if grouped else ([0], [])
    args = [t.cuda() for t in (query, k, v, torch.tensor(starts, dtype=torch.int32),
                               torch.tensor(prefix, dtype=torch.int32), tables, torch.tensor(lengths, dtype=torch.int32))]
    got = cf.paged_attention_shared(*args).cpu().double()
    half = torch.finfo(torch.bfloat16).eps / 2
    for s, last in enumerate((block - 4096, block - 4096, 0)):
        keys, values = (torch.cat([x[1, :, 0], x[0, :last, 0]]).double() for x in (k, v))
        p = torch.softmax(query[s].double() @ keys.T * dim**-0.5, -1)
        ref, size = p @ values, p @ values.abs()
        # As shared_util.check, with the tokens that the table names.
        tolerance = (2.0**-16 + 2.0**-24 * len(keys) / 32 + half) * size + half * ref.abs()
        assert ((got[s] - ref).abs() <= tolerance).all()
