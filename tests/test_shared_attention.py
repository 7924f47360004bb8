"""Attention behind shared prompts on the CPU: definition and refusals."""

from __future__ import annotations

import ctypes

import pytest
import torch

import cuda_force_amd as cf
from cuda_force_amd import _lib
from cuda_force_amd.paged_cache import _paged_attention_reference
from tests.shared_util import build, check


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("block", [1, 5, 16])
def test_definition(dtype, block):
    c = build([(20, [20, 25, 3]), (7, [0, 9])], 4, 2, 16, block, dtype, loners=2)
    check(cf.paged_attention_shared(*c.args("cpu")), c)
    check(_paged_attention_reference(c.query, c.k, c.v, c.tables, c.context, c.scale), c)


def test_an_entry_that_names_no_page_and_a_context_past_the_table():
    c = build([(8, [10, 12])], 2, 1, 8, 4, torch.float32)
    c.tables[1, 0] = 1000
    c.tables[0, 1] = -1
    check(cf.paged_attention_shared(*c.args("cpu")), c)
    c.context[1] = 100
    c.context[0] = -5
    c.k[torch.isnan(c.k)] = 0.0
    c.v[torch.isnan(c.v)] = 0.0
    check(cf.paged_attention_shared(*c.args("cpu")), c)


def test_default_scale_and_gradients_through_the_composition():
    c = build([(8, [10, 12])], 2, 1, 8, 4, torch.float32)
    a = cf.paged_attention_shared(*c.args("cpu")[:-1])
    assert torch.equal(a, cf.paged_attention_shared(*c.args("cpu")))
    q = c.query.clone().requires_grad_(True)
    cf.paged_attention_shared(q, *c.args("cpu")[1:]).sum().backward()
    assert torch.isfinite(q.grad).all()


def test_refusals():
    c = build([(8, [10, 12])], 2, 1, 8, 4, torch.float32)
    names = ["query", "k", "v", "starts", "prefix", "tables", "context"]

    def call(**changed):
        values = dict(zip(names, c.args("cpu")))
        values.update(changed)
        return cf.paged_attention_shared(*values.values())

    call()
    for changed in ({"query": c.query[0]}, {"v": c.v[:1]}, {"k": c.k[..., :4], "v": c.v[..., :4]},
                    {"query": torch.zeros(2, 3, 8), "k": torch.zeros(4, 4, 2, 8), "v": torch.zeros(4, 4, 2, 8)},
                    {"k": c.k.transpose(0, 1), "v": c.v.transpose(0, 1)}, {"tables": c.tables[:1]},
                    {"context": c.context[:1]}, {"starts": c.starts[:1]}, {"prefix": c.prefix[None]},
                    {"k": c.k.to(torch.bfloat16), "v": c.v.to(torch.bfloat16)},
                    {"query": torch.zeros(2, 2, 1025), "k": torch.zeros(4, 4, 1, 1025),
                     "v": torch.zeros(4, 4, 1, 1025)}):
        with pytest.raises(ValueError):
            call(**changed)
    for name in ("starts", "prefix", "tables", "context"):
        with pytest.raises(TypeError):
            call(**{name: getattr(c, name).long()})


def test_c_abi_refusals_before_any_launch():
    lib = _lib.load()
    fake, null = ctypes.c_void_p(0x1000), ctypes.c_void_p(0)

    def call(query=fake, k=fake, starts=fake, tables=fake, out=fake, dtype=_lib.CF_BF16, pages=100, sequences=4,
             groups=1, heads=8, kv_heads=2, dim=64, block=16, width=10, ws=fake, ws_bytes=1 << 30):
        return lib.cf_paged_attention_shared(query, k, fake, starts, fake, tables, fake, out, dtype, pages, sequences,
                                             groups, heads, kv_heads, dim, block, width, 1.0, ws, ws_bytes, null)

    assert call(sequences=0) == _lib.CF_OK
    for case in ({"query": null}, {"k": null}, {"starts": null}, {"tables": null}, {"out": null}, {"dtype": 9},
                 {"pages": 0}, {"groups": -1}, {"kv_heads": 3}, {"kv_heads": 0}, {"dim": 1025}, {"block": 0},
                 {"width": 0}, {"ws": null}, {"ws_bytes": 8}, {"ws": ctypes.c_void_p(0x1008)},
                 {"query": ctypes.c_void_p(0x1001)}, {"pages": 2**27, "block": 16}, {"sequences": 2**29},
                 {"groups": 2**21}):
        assert call(**case) == _lib.CF_ERR_INVALID_ARGUMENT, case
    size = lib.cf_paged_attention_shared_workspace_bytes
    assert size(_lib.CF_BF16, 4, 1, 8, 2, 64, 16, 10) > 0
    assert size(_lib.CF_BF16, 4, 1, 8, 3, 64, 16, 10) == 0
    # 128 sequences of 32 heads over 32768 shared tokens: tens of MB, not GB.
    assert size(_lib.CF_BF16, 128, 1, 32, 8, 128, 32, 1040) < 64e6


def test_more_rows_than_a_launch_takes_are_refused_before_any():
    lib = _lib.load()
    fake, null = ctypes.c_void_p(0x1000), ctypes.c_void_p(0)

    def call(sequences, heads, kv_heads, dim):
        return lib.cf_paged_attention_shared(fake, fake, fake, null, null, fake, fake, fake, _lib.CF_BF16, 100,
                                             sequences, 0, heads, kv_heads, dim, 16, 1, 1.0, fake, 2**62, null)

    bad = _lib.CF_ERR_INVALID_ARGUMENT
    assert call(2**23, 32, 32, 64) == bad     # a wave a rest: 2^26 workgroups
    assert call(2**22, 32, 2, 64) == bad      # rows to join, a wave each: 2^25
    assert call(2**20, 17, 1, 300) == bad     # rows to join, a workgroup each
    assert b"too many" in lib.cf_last_error()
