"""Storing into a paged cache from tensors that share memory with it."""

from __future__ import annotations

import ctypes

import pytest
import torch

import cuda_force_amd as cf
from cuda_force_amd import _lib

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def cache(device, dtype=torch.float32, tokens=4000, heads=2, dim=64):
    gen = torch.Generator().manual_seed(0)
    return [torch.randn(tokens // 16, 16, heads, dim, generator=gen).to(dtype).to(device) for _ in range(2)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_the_cache_itself_are_read_before_any_is_written(device, dtype):
    """Tokens moved within a cache: every one to the place of the next."""
    k, v = cache(device, dtype)
    n = k.shape[0] * 16
    slots = (torch.arange(n, device=device) + 1) % n
    want = [t.view(n, 2, 64).roll(1, 0).clone() for t in (k, v)]
    cf.cache_write(k.view(n, 2, 64), v.view(n, 2, 64), k, v, slots)
    assert torch.equal(k.view(n, 2, 64), want[0]) and torch.equal(v.view(n, 2, 64), want[1])
    # Crosswise: what is given as values lies where keys are written.
    k, v = cache(device, dtype)
    want = [v.view(n, 2, 64).flip(0).clone(), k.view(n, 2, 64).flip(0).clone()]
    cf.cache_write(v.view(n, 2, 64), k.view(n, 2, 64), k, v, torch.arange(n, device=device).flip(0))
    assert torch.equal(k.view(n, 2, 64), want[0]) and torch.equal(v.view(n, 2, 64), want[1])
    # A part of it, read with strides.
    k, v = cache(device, dtype)
    given = [t.view(n, 2, 64)[::3].clone() for t in (k, v)]
    slots = torch.randperm(n)[: len(given[0])].to(device)
    want = [t.clone() for t in (k, v)]
    for t, x in zip(want, given):
        t.view(n, 2, 64)[slots] = x
    cf.cache_write(k.view(n, 2, 64)[::3], v.view(n, 2, 64)[::3], k, v, slots)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


@pytest.mark.parametrize("device", DEVICES)
def test_caches_that_share_memory_are_refused(device):
    x = torch.randn(4, 2, 64, device=device)
    slots = torch.arange(4, device=device)
    both = torch.zeros(6, 16, 2, 64, device=device)
    codes = torch.zeros(6, 16, 2, 64, dtype=torch.int8, device=device)
    scales = torch.zeros(7, 16, 2, device=device)
    for call in (lambda: cf.cache_write(x, x, both[:4], both[2:], slots),
                 lambda: cf.cache_write(x, x, codes[:4], codes[2:], slots, scales[:4], scales[3:]),
                 lambda: cf.cache_write(x, x, codes[:3], codes[3:], slots, scales[:3], scales[2:5])):
        with pytest.raises((RuntimeError, ValueError)):
            call()
    assert (both == 0).all() and (codes == 0).all() and (scales == 0).all()
    cf.cache_write(x, x, both[:3], both[3:], slots)  # neighbours do not share any
    cf.cache_write(x, x, codes[:3], codes[3:], slots, scales[:3], scales[3:6])
    assert (both.view(6, 16, 2, 64)[:, 4:] == 0).all()


def test_c_abi_refuses_shared_memory_before_any_launch():
    lib = _lib.load()
    null = ctypes.c_void_p(0)
    at = ctypes.c_void_p

    def write(k=0x100000, v=0x200000, ks=0x300000, vs=0x400000, x=0x500000, y=0x600000, form=_lib.CF_CACHE_INT8):
        # 4 tokens of 2 heads of 64 in bf16 to 32 slots: 1 KiB given each, 4 KiB of codes, 256 bytes of scales.
        return lib.cf_cache_write(at(x), at(y), _lib.CF_BF16, 4, 2, 64, 128, 64, 128, 64, at(0x700000), at(k), at(v),
                                  form, at(ks), at(vs), 32, null)

    for case in ({"v": 0x100000 + 4080}, {"v": 0x100000 - 16}, {"vs": 0x300000 + 252}, {"x": 0x100000 + 4080},
                 {"x": 0x200000 - 16}, {"y": 0x100000}, {"y": 0x200000 + 16}, {"y": 0x300000}, {"x": 0x400000 + 240},
                 {"k": 0x400000}, {"form": _lib.CF_CACHE_PLAIN, "v": 0x100000 + 8176}):
        assert write(**case) == _lib.CF_ERR_INVALID_ARGUMENT, case
