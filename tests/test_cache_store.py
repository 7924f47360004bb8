"""Storing into a paged cache and reading back on the CPU: definition, refusals."""

from __future__ import annotations

import ctypes

import pytest
import torch

import cuda_force_amd as cf
from cuda_force_amd import _lib
from tests import codes_util

CODES = [torch.int8, torch.float8_e4m3fn]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def caches(pages, block, heads, dim, dtype):
    k = torch.zeros(pages, block, heads, dim).to(dtype)
    s = torch.ones(pages, block, heads) if dtype in CODES else None
    return k, k.clone(), s, None if s is None else s.clone()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("codes", CODES)
def test_codes_are_the_nearest_ones(dtype, codes):
    x = codes_util.hard_rows(dtype).view(24, 1, 64)
    k, v, ks, vs = caches(6, 4, 1, 64, codes)
    cf.cache_write(x, -x, k, v, torch.arange(24), ks, vs)
    numbers, scales = codes_util.rows(x, codes)
    assert torch.equal(k.float().view(24, 1, 64).double(), numbers)
    assert torch.equal(v.float().view(24, 1, 64).double(), -numbers)
    for s in (ks, vs):
        assert torch.equal(s.view(24, 1).nan_to_num(7.0), scales.nan_to_num(7.0))
    back, _ = cf.cache_read(k, v, torch.arange(24), ks, vs)
    want = (numbers * scales.double().unsqueeze(-1)).float()
    assert torch.equal(back.nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [*DTYPES, *CODES])
def test_slots(dtype):
    given = torch.bfloat16 if dtype in CODES else dtype
    k, v, ks, vs = caches(3, 4, 2, 16, dtype)
    x = torch.randn(7, 2, 16).to(given)
    slots = torch.tensor([3, -1, 12, 11, 3, 0, 2**40])  # out of range, and one twice
    before = k.clone().view(12, 2, 16)
    cf.cache_write(x, 2 * x, k, v, slots, ks, vs)
    keys, values = cf.cache_read(k, v, slots, ks, vs, dtype=given)
    alone = caches(3, 4, 2, 16, dtype)
    cf.cache_write(x, 2 * x, alone[0], alone[1], torch.tensor([1, 2, 4, 5, 6, 7, 8]), *alone[2:])
    one, two = cf.cache_read(alone[0], alone[1], torch.tensor([1, 2, 4, 5, 6, 7, 8]), *alone[2:], dtype=given)
    one[0], two[0] = one[4], two[4]  # the later token of slot 3
    for i in (1, 2, 6):
        one[i], two[i] = 0, 0
    assert torch.equal(keys, one) and torch.equal(values, two)
    untouched = [s for s in range(12) if s not in (0, 3, 11)]
    assert torch.equal(k.float().view(12, 2, 16)[untouched], before.float()[untouched])


def test_views_of_a_projection_and_empty_calls():
    fused = torch.randn(5, 6, 8)
    k, v, _, _ = caches(2, 4, 2, 8, torch.float32)
    cf.cache_write(fused[:, 2:4], fused[:, 4:], k, v, torch.arange(5))
    assert torch.equal(k.view(8, 2, 8)[:5], fused[:, 2:4]) and torch.equal(v.view(8, 2, 8)[:5], fused[:, 4:])
    cf.cache_write(fused[:0, 2:4], fused[:0, 4:], k, v, torch.arange(0))
    keys, values = cf.cache_read(k, v, torch.arange(0))
    assert keys.shape == values.shape == (0, 2, 8)


def test_refusals():
    x = torch.randn(4, 2, 8)
    k, v, ks, vs = caches(2, 4, 2, 8, torch.int8)
    plain = torch.zeros(2, 4, 2, 8)
    slots = torch.arange(4)

    def write(error, x=x, values=None, k=k, v=v, slots=slots, ks=ks, vs=vs):
        with pytest.raises(error):
            cf.cache_write(x, x if values is None else values, k, v, slots, ks, vs)

    write(ValueError, x=x[:3])
    write(ValueError, values=x[:, :1])
    write(ValueError, v=v[:1])
    write(ValueError, k=k.transpose(0, 1), v=v.transpose(0, 1))
    write(ValueError, ks=None)
    write(ValueError, ks=ks[:1])
    write(ValueError, k=plain, v=plain)
    write(ValueError, slots=slots.view(2, 2))
    write(ValueError, x=x.clone().requires_grad_(True))
    write(ValueError, v=k)
    write(ValueError, vs=ks)
    write(TypeError, slots=slots.int())
    write(TypeError, ks=ks.double())
    write(TypeError, values=x.double())
    write(TypeError, k=k.int(), v=v.int())
    write(TypeError, k=plain.double(), v=plain.double(), ks=None, vs=None)
    with pytest.raises(ValueError):
        cf.cache_read(plain, plain, slots, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        cf.cache_read(k, v, slots)
    with pytest.raises(TypeError):
        cf.cache_read(k, v, slots.int(), ks, vs)


def test_c_abi_refusals_before_any_launch():
    lib = _lib.load()
    fake, null, other = ctypes.c_void_p(0x1000), ctypes.c_void_p(0), ctypes.c_void_p(0x2000)

    def write(x=fake, dtype=_lib.CF_BF16, tokens=4, heads=2, dim=64, slots=fake, cache=fake, form=_lib.CF_CACHE_INT8,
              scales=fake, num_slots=100):
        return lib.cf_cache_write(x, fake, dtype, tokens, heads, dim, 128, 64, 128, 64, slots, cache, other, form,
                                  scales, other, num_slots, null)

    def read(x=fake, dtype=_lib.CF_BF16, tokens=4, heads=2, dim=64, slots=fake, cache=fake, form=_lib.CF_CACHE_INT8,
             scales=fake, num_slots=100):
        return lib.cf_cache_read(cache, fake, form, scales, fake, num_slots, slots, tokens, heads, dim, x, fake, dtype,
                                 null)

    for call in (write, read):
        assert call(tokens=0) == call(heads=0) == call(dim=0) == _lib.CF_OK
        for case in ({"x": null}, {"dtype": 9}, {"form": 7}, {"slots": null}, {"cache": null}, {"scales": null},
                     {"num_slots": -1}, {"num_slots": 2**31}, {"heads": 2**15}, {"x": ctypes.c_void_p(0x1001)},
                     {"scales": ctypes.c_void_p(0x1002)}, {"slots": ctypes.c_void_p(0x1004)},
                     {"tokens": 2**40}):
            assert call(**case) == _lib.CF_ERR_INVALID_ARGUMENT, case
    # One place for keys and values.
    assert write(cache=other) == write(scales=other) == _lib.CF_ERR_INVALID_ARGUMENT
