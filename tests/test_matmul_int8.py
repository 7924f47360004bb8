"""Row-wise int8 and the products of it on the CPU: definition, refusals."""

from __future__ import annotations

import ctypes

import pytest
import torch

import cuda_force_amd as cf
from cuda_force_amd import _lib
from tests import codes_util

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_by_their_definition(dtype):
    x = codes_util.hard_rows(dtype)
    codes, scales = cf.quantize_int8_rows(x)
    numbers, want = codes_util.rows(x, torch.int8)
    assert codes.dtype == torch.int8 and torch.equal(codes.double(), numbers)
    assert torch.equal(scales.nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_products(dtype):
    gen = torch.Generator().manual_seed(0)
    x = torch.randint(-128, 128, (2, 3, 40), generator=gen, dtype=torch.int8)
    w = torch.randint(-128, 128, (7, 40), generator=gen, dtype=torch.int8)
    xs, ws = torch.rand(2, 3, generator=gen), torch.rand(7, generator=gen)
    bias = torch.randn(7, generator=gen).to(dtype)
    y = cf.matmul_int8(x, w, xs, ws, bias=bias, dtype=dtype)
    want = (x.long() @ w.long().t()).double() * xs.double().unsqueeze(-1) * ws.double() + bias.double()
    assert y.dtype == dtype and y.shape == (2, 3, 7)
    # One rounding to the type, and fp32's of two products, a sum and the
    # conversion, relative to what they round.
    size = want.abs() + bias.double().abs()
    assert ((y.double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 5 * 2.0**-24 * size).all()


def test_empty_and_padded():
    codes, scales = cf.quantize_int8_rows(torch.zeros(0, 8))
    assert codes.shape == (0, 8) and scales.shape == (0,)
    codes, scales = cf.quantize_int8_rows(torch.zeros(3, 0))
    assert codes.shape == (3, 0) and torch.equal(scales, torch.ones(3))
    wide = torch.randn(4, 20)
    assert torch.equal(cf.quantize_int8_rows(wide[:, :12])[0], cf.quantize_int8_rows(wide[:, :12].clone())[0])
    y = cf.matmul_int8(torch.zeros(3, 0, dtype=torch.int8), torch.zeros(5, 0, dtype=torch.int8), torch.ones(3),
                       torch.ones(5), dtype=torch.float32)
    assert torch.equal(y, torch.zeros(3, 5))


def test_refusals():
    x, w = torch.ones(3, 8, dtype=torch.int8), torch.ones(5, 8, dtype=torch.int8)
    xs, ws = torch.ones(3), torch.ones(5)

    def call(error, x=x, w=w, xs=xs, ws=ws, bias=None, dtype=torch.bfloat16):
        with pytest.raises(error):
            cf.matmul_int8(x, w, xs, ws, bias=bias, dtype=dtype)

    call(TypeError, x=x.int())
    call(TypeError, w=w.float())
    call(TypeError, xs=xs.double())
    call(TypeError, bias=torch.ones(5))
    call(ValueError, w=w[:, :4])
    call(ValueError, xs=xs[:2])
    call(ValueError, ws=ws[:2])
    call(ValueError, bias=torch.ones(4, dtype=torch.bfloat16))
    big = torch.ones(1, 131072, dtype=torch.int8)
    call(ValueError, x=big, w=big, xs=torch.ones(1), ws=torch.ones(1))
    with pytest.raises(ValueError):
        cf.quantize_int8_rows(torch.tensor(1.0))


def test_c_abi_refusals_before_any_launch():
    lib = _lib.load()
    fake, null = ctypes.c_void_p(0x1000), ctypes.c_void_p(0)

    def rows(x=fake, dtype=_lib.CF_BF16, n=4, cols=64, stride=64, codes=fake, scales=fake):
        return lib.cf_quantize_int8_rows(x, dtype, n, cols, stride, codes, scales, null)

    assert rows(n=0) == rows(cols=0) == _lib.CF_OK
    for case in ({"x": null}, {"codes": null}, {"scales": null}, {"dtype": 5}, {"stride": 63},
                 {"x": ctypes.c_void_p(0x1001)}, {"scales": ctypes.c_void_p(0x1002)}):
        assert rows(**case) == _lib.CF_ERR_INVALID_ARGUMENT, case

    def product(x=fake, w=fake, xs=fake, ws=fake, bias=null, y=fake, dtype=_lib.CF_BF16, m=4, n=8, k=64):
        return lib.cf_matmul_int8(x, w, xs, ws, bias, y, dtype, m, n, k, null)

    assert product(m=0) == product(n=0) == _lib.CF_OK
    for case in ({"x": null}, {"w": null}, {"xs": null}, {"ws": null}, {"y": null}, {"dtype": 5}, {"k": 131072},
                 {"k": -1}, {"m": 2**31}, {"bias": ctypes.c_void_p(0x1001)}, {"y": ctypes.c_void_p(0x1001)},
                 {"m": 2**28, "n": 2**20}):
        assert product(**case) == _lib.CF_ERR_INVALID_ARGUMENT, case
