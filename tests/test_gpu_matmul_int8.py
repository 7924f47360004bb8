"""Row-wise int8 and the products of it on the GPU."""

from __future__ import annotations

import pytest
import torch

import cuda_force_amd as cf
from cuda_force_amd.ops import _nearest_codes
from tests import codes_util

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def rows(x):
    codes, scales = cf.quantize_int8_rows(x.cuda())
    want, want_scales = _nearest_codes(x, torch.int8)
    assert torch.equal(codes.cpu(), want)
    assert torch.equal(scales.cpu().nan_to_num(7.0), want_scales.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_hard_rows(dtype):
    for cols in (8, 64, 100, 1024, 4096):
        rows(codes_util.hard_rows(dtype, cols))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 7, 8, 512, 1000, 2048, 4100, 8192, 11008, 20000, 40000, 65536, 70000])
def test_row_lengths(dtype, cols):
    rows((torch.randn(5, cols) * torch.exp(torch.randn(5, 1))).to(dtype))
    if cols <= 8192:
        rows((torch.randn(2100, cols) * torch.exp(torch.randn(2100, 1))).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_padded_and_misaligned_rows(dtype):
    wide = torch.randn(30, 300).to(dtype)
    for part in (wide[:, :256], wide[:, 1:257], wide[::3, 8:72], wide.t(), wide[:1].expand(9, 300)):
        rows(part)
    on_gpu = wide.cuda()
    assert torch.equal(cf.quantize_int8_rows(on_gpu[:, 3:67])[0].cpu(), _nearest_codes(wide[:, 3:67], torch.int8)[0])


def product(m, n, k, dtype, bias=True, seed=0, misaligned=False):
    gen = torch.Generator().manual_seed(seed)
    x, w = (torch.randint(-128, 128, (r, k), generator=gen, dtype=torch.int8) for r in (m, n))
    xs, ws = (torch.rand(r, generator=gen) * 1e-2 for r in (m, n))
    b = torch.randn(n, generator=gen).to(dtype) if bias else None
    if misaligned:
        flat = torch.empty(m * k + 1, dtype=torch.int8, device="cuda")
        x_gpu = flat[1:].view(m, k).copy_(x)
    else:
        x_gpu = x.cuda()
    args = [x_gpu, w.cuda(), xs.cuda(), ws.cuda()]
    y = cf.matmul_int8(*args, bias=None if b is None else b.cuda(), dtype=dtype)
    again = cf.matmul_int8(*args, bias=None if b is None else b.cuda(), dtype=dtype)
    assert torch.equal(y, again)
    # Sums by fp64 on the GPU: exact.
    sums = x.cuda().double() @ w.cuda().double().t()
    want = sums * xs.cuda().double()[:, None] * ws.cuda().double()
    size = want.abs()
    if b is not None:
        want = want + b.cuda().double()
        size = size + b.cuda().double().abs()
    tolerance = torch.finfo(dtype).eps / 2 * want.abs() + 5 * 2.0**-24 * size
    if dtype == torch.float16:
        tolerance = tolerance + 2.0**-25  # half of fp16's smallest number
    assert y.shape == (m, n) and y.dtype == dtype
    assert ((y.double() - want).abs() <= tolerance).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 5, 16, 17, 33, 64, 65, 100, 300])
@pytest.mark.parametrize("n,k", [(16, 64), (100, 16), (33, 1008), (512, 528), (1030, 4096)])
def test_sizes(dtype, m, n, k):
    product(m, n, k, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(2048, 4096, 256), (2049, 4099, 144), (5000, 2600, 1040), (700, 1500, 4096),
                                   (4096, 4096, 128), (260, 8192, 11008), (9000, 300, 512), (2560, 5120, 400)])
def test_large_tiles(dtype, m, n, k):
    product(m, n, k, dtype, bias=n % 2 == 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(17, 8200, 400), (64, 8200, 128), (40, 8250, 16), (200, 4000, 2064), (333, 4096, 144),
                                   (333, 4100, 4112), (500, 2600, 1040), (640, 4096, 272), (128, 11008, 1152)])
def test_middling_products(dtype, m, n, k):
    """Tiles of 64 and 96 rows, one or two groups of waves on a tile's k (of as
    many stages, of one more, of a single one)."""
    product(m, n, k, dtype)


@pytest.mark.parametrize("m,n,k", [(3, 5, 1), (20, 30, 7), (65, 70, 100), (130, 40, 1001), (4, 4, 131071)])
def test_any_depth(m, n, k):
    for dtype in DTYPES:
        product(m, n, k, dtype)


def test_no_products():
    for m, n in ((1, 5), (40, 300), (333, 4100), (2100, 4096)):
        product(m, n, 0, torch.bfloat16, bias=False)
        product(m, n, 0, torch.float32)


def test_the_longest_sums():
    product(17, 40, 131056, torch.float32, bias=False)
    product(300, 260, 131056, torch.float32, bias=False)
    x = torch.full((70, 131056), -128, dtype=torch.int8, device="cuda")
    y = cf.matmul_int8(x, x[:64], torch.ones(70, device="cuda"), torch.ones(64, device="cuda"), dtype=torch.float32)
    assert (y == 128.0 * 128.0 * 131056).all()


def test_misaligned_operands_and_leading_dimensions():
    product(70, 48, 64, torch.bfloat16, misaligned=True)
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(2, 7, 96, generator=gen)
    w = torch.randn(40, 96, generator=gen)
    sets = []
    for device in ("cpu", "cuda"):
        codes, scales = cf.quantize_int8_rows(x.to(device))
        wc, ws = cf.quantize_int8_rows(w.to(device))
        sets.append(cf.matmul_int8(codes, wc, scales, ws, dtype=torch.float32).cpu())
    assert sets[1].shape == (2, 7, 40)
    assert (sets[0] - sets[1]).abs().max() <= 4 * 2.0**-24 * sets[0].abs().max()


def test_a_row_that_is_not_finite_gives_nan_alone():
    x = torch.randn(70, 256)
    x[3, 9], x[40, 0] = float("inf"), float("nan")
    codes, scales = cf.quantize_int8_rows(x.cuda())
    w, ws = cf.quantize_int8_rows(torch.randn(128, 256).cuda())
    bad = torch.isnan(cf.matmul_int8(codes, w, scales, ws)).cpu()
    assert bad[[3, 40]].all() and bad.sum() == 2 * 128


@pytest.mark.parametrize("m", [3, 200, 2048])
def test_graph(m):
    x = torch.randn(m, 512, device="cuda", dtype=torch.bfloat16)
    w, ws = cf.quantize_int8_rows(torch.randn(4096, 512, device="cuda"))

    def step():
        codes, scales = cf.quantize_int8_rows(x)
        return cf.matmul_int8(codes, w, scales, ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, step())


def test_results_and_rows_past_2_to_the_31():
    m, n, k = 70000, 40000, 16
    x = torch.randint(-128, 128, (m, k), device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), device="cuda", dtype=torch.int8)
    ones = torch.ones(m, device="cuda")
    y = cf.matmul_int8(x, w, ones, ones[:n])
    for at in (0, 53687, 53688, m - 1):  # 2^31 / n lies between the middle two
        want = (x[at].double() @ w.double().t()).to(torch.bfloat16)
        assert torch.equal(y[at], want)
    del y
    rows = 2**31 // 8192 + 9
    x = torch.randn(rows, 8192, device="cuda", dtype=torch.bfloat16)
    codes, scales = cf.quantize_int8_rows(x)
    for at in (0, rows - 10, rows - 9, rows - 1):
        want, want_scales = _nearest_codes(x[at : at + 1].cpu(), torch.int8)
        assert torch.equal(codes[at : at + 1].cpu(), want) and torch.equal(scales[at : at + 1].cpu(), want_scales)
    del x, codes
    torch.cuda.empty_cache()
