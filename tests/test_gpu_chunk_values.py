"""Attention of chunks over values of every kind, against float64: small ones in
caches of codes, whose weights keep their bits whatever else a row meets, and
ones that are not finite."""

from __future__ import annotations

import pytest
import torch

import cuda_force_amd as cf
from tests.chunk_util import CODES, build, check, reference

pytestmark = pytest.mark.gpu
# Few rows a tile, some more, and many (tiles of 32, 64 and 128 rows).
ROWS = [[(1, 700), (1, 1100)], [(9, 500), (5, 300)], [(60, 700), (40, 200)], [(300, 900)]]


def small(sequences, dtype, held, dim=128, heads=4, kv_heads=1, size=1e-8):
    c = build(sequences, heads, kv_heads, dim, 16, dtype, held)
    c.v_scales = c.v_scales * size
    return c


def run(c):
    check(cf.paged_attention_chunk(*c.args()), c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("held", CODES)
@pytest.mark.parametrize("sequences", ROWS)
@pytest.mark.parametrize("dim", [64, 128, 256, 80])
def test_small_values_behind_pages_left_out(dtype, held, sequences, dim):
    """Steps in which a row meets no token: none, the first ones, and some later."""
    c = small(sequences, dtype, held, dim)
    run(c)
    c.tables[:, :8] = -1
    run(c)
    c = small(sequences, dtype, held, dim)
    c.tables[:, 4:12] = -1
    run(c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("held", CODES)
@pytest.mark.parametrize("sequences", ROWS)
@pytest.mark.parametrize("dim", [64, 128, 256, 80])
def test_small_values_beside_rows_of_zeros(dtype, held, sequences, dim):
    """Rows of zeros have the scale 1, far above the others': alone in the first
    steps, among others in one, as tokens of both halves of a step, and (in e4m3)
    with codes of -0."""
    zeros = [range(0, 200), [3], [350, 351, 420, 470], range(500, 540)]
    for places in zeros:
        c = small(sequences, dtype, held, dim)
        for s, length in enumerate(c.context.tolist()):
            for t in places:
                if t < length:
                    page, at = int(c.tables[s, t // 16]), t % 16
                    c.v[page, at] = 0
                    if held == torch.float8_e4m3fn:
                        c.v.view(torch.uint8)[page, at, :, ::3] = 0x80
                    c.v_scales[page, at] = 1.0
        run(c)


@pytest.mark.parametrize("held", CODES)
@pytest.mark.parametrize("sequences", ROWS)
def test_a_scale_of_1_that_is_no_row_of_zeros(held, sequences):
    """Small values next to tokens whose values are up to the largest code times 1."""
    c = small(sequences, torch.float32, held)
    for s, length in enumerate(c.context.tolist()):
        for t in (2, 40, length - 1):
            page, at = int(c.tables[s, t // 16]), t % 16
            c.v[page, at] = 0
            c.v[page, at, :, t % 128] = 1.0
            c.v_scales[page, at] = 1.0
    run(c)


def not_finite(c, s, t, dims, bad):
    """Values of token t of sequence s, of all its heads."""
    page, at = int(c.tables[s, t // 16]), t % 16
    if c.v_scales is None:
        c.v[page, at][:, dims] = bad
    else:
        c.v.view(torch.uint8)[page, at][:, dims] = 0x7F if bad > 0 else 0xFF


@pytest.mark.parametrize("dtype,held", [(torch.float32, None), (torch.bfloat16, None), (torch.float16, None),
                                        (torch.float32, CODES[1]), (torch.bfloat16, CODES[1])])
@pytest.mark.parametrize("sequences", [*ROWS, [(100, 100), (3, 100), (40, 300), (1, 17)]])
@pytest.mark.parametrize("dim", [64, 128, 256, 80, 20])
def test_values_that_are_not_finite_reach_their_own_dims_alone(dtype, held, sequences, dim):
    """Of tokens that some rows of a step see and others do not, and of tokens
    that all of them see: infinities keep their signs, two of them give NaN."""
    c = build(sequences, 4, 1, dim, 16, dtype, held)
    for s, (new, length) in enumerate(sequences):
        for t in {0, length - new, length - new // 2 - 1, length - 1}:
            not_finite(c, s, t, [1, dim - 1], float("inf"))
        not_finite(c, s, length - new // 3 - 1, [dim - 1, dim - 2], -float("inf"))
        if held is None:
            not_finite(c, s, length - new // 4 - 1, [5], float("nan"))
    got = cf.paged_attention_chunk(*c.args()).cpu()
    want, _ = reference(c)
    assert (~torch.isfinite(want)).any() and torch.isfinite(want).any()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isposinf(got), torch.isposinf(want))
    assert torch.equal(torch.isneginf(got), torch.isneginf(want))
    # The others as without them: dims do not meet.
    bits = c.v if held is None else c.v.view(torch.uint8)
    bits[~torch.isfinite(c.v.float())] = 0
    clean = cf.paged_attention_chunk(*c.args()).cpu()
    finite = torch.isfinite(want)
    assert torch.equal(got[finite], clean[finite])
    check(clean, c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("held", CODES)
@pytest.mark.parametrize("sequences", ROWS)
def test_scales_of_1_throughout(dtype, held, sequences):
    """A cache of codes without scales of their own, some rows of zeros at first and later."""
    c = build(sequences, 4, 1, 64, 16, dtype, held)
    c.k_scales[c.k_scales.isfinite()] = 1.0
    c.v_scales[c.v_scales.isfinite()] = 1.0
    c.scale = 1e-3
    for s, length in enumerate(c.context.tolist()):
        for t in [*range(70), *range(130, 135), length - 1]:
            c.v[int(c.tables[s, t // 16]), t % 16] = 0
    run(c)
