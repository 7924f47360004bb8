"""Attention of chunks over caches of codes whose values are small, against
float64: a row's weights keep their bits whatever else it meets."""

from __future__ import annotations

import pytest
import torch

import cuda_force_amd as cf
from tests.chunk_util import CODES, build, check

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
