"""Operators of serving in 8 bits at sizes past 32 bits and past one launch."""

from __future__ import annotations

import pytest
import torch

import cuda_force_amd as cf

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
