"""Attention of chunks of new tokens on the CPU: definition and refusals."""

from __future__ import annotations

import ctypes

import pytest
import torch

import cuda_force_amd as cf
from cuda_force_amd import _lib
from tests.chunk_util import CODES, build, check

CASES = [(3, 20), (1, 17), (0, 9), (5, 5), (1, 1), (2, 0), (4, 2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("held", [None, *CODES])
@pytest.mark.parametrize("block", [1, 5, 16])
def test_definition(dtype, held, block):
    c = build(CASES, 4, 2, 16, block, dtype, held, before=2, behind=3)
    got = cf.paged_attention_chunk(*c.args("cpu"))
    check(got, c)
    assert (got[:2] == 0).all() and (got[-3:] == 0).all()


def test_starts_tables_and_lengths_as_stored_wrongly():
    c = build([(4, 10), (6, 12), (3, 8)], 2, 1, 8, 4, torch.float32, bad=False)
    c.tables[1, 0] = 1000
    c.tables[0, 1] = -1
    check(cf.paged_attention_chunk(*c.args("cpu")), c)
    c.context[2] = 100
    c.context[0] = -5
    check(cf.paged_attention_chunk(*c.args("cpu")), c)
    for starts in ([5, 2, 9, 1], [-3, 4, 4, 100], [13, 13, 13, 13]):
        c.starts = torch.tensor(starts, dtype=torch.int32)
        check(cf.paged_attention_chunk(*c.args("cpu")), c)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_stays_out(bad):
    c = build([(6, 20)], 2, 1, 8, 4, torch.float32)
    clean = cf.paged_attention_chunk(*c.args("cpu"))
    page, at = int(c.tables[0, 17 // 4]), 17 % 4  # row 3's own token
    c.k[page, at], c.v[page, at] = bad, bad
    got = cf.paged_attention_chunk(*c.args("cpu"))
    assert torch.equal(got[:3], clean[:3]) and not torch.isfinite(got[3:]).all(-1).any()


def test_default_scale_and_gradients_through_the_composition():
    c = build([(3, 10), (1, 12)], 2, 1, 8, 4, torch.float32)
    a = cf.paged_attention_chunk(*c.args("cpu")[:-1])
    assert torch.equal(a, cf.paged_attention_chunk(*c.args("cpu")))
    q = c.query.clone().requires_grad_(True)
    cf.paged_attention_chunk(q, *c.args("cpu")[1:]).sum().backward()
    assert torch.isfinite(q.grad).all()


def test_refusals():
    plain = build([(3, 10), (1, 12)], 2, 1, 8, 4, torch.float32)
    codes = build([(3, 10), (1, 12)], 2, 1, 8, 4, torch.float32, torch.int8)
    names = ["query", "k", "v", "starts", "tables", "context", "ks", "vs"]

    def call(c, **changed):
        values = dict(zip(names, c.args("cpu")))
        values.update(changed)
        return cf.paged_attention_chunk(*values.values())

    call(plain)
    call(codes)
    c = plain
    for changed in ({"query": c.query[0]}, {"v": c.v[:1]}, {"k": c.k[..., :4], "v": c.v[..., :4]},
                    {"query": torch.zeros(4, 3, 8), "k": torch.zeros(4, 4, 2, 8), "v": torch.zeros(4, 4, 2, 8)},
                    {"k": c.k.transpose(0, 1), "v": c.v.transpose(0, 1)}, {"tables": c.tables[:1]},
                    {"context": c.context[:1]}, {"starts": c.starts[:1]}, {"starts": c.starts[None]},
                    {"k": c.k.to(torch.bfloat16), "v": c.v.to(torch.bfloat16)}, {"ks": codes.k_scales},
                    {"query": torch.zeros(4, 2, 1025), "k": torch.zeros(4, 4, 1, 1025),
                     "v": torch.zeros(4, 4, 1, 1025)}):
        with pytest.raises(ValueError):
            call(c, **changed)
    for changed in ({"ks": None}, {"vs": None}, {"ks": codes.k_scales[:1]}, {"v": codes.v.view(torch.float8_e4m3fn)}):
        with pytest.raises(ValueError):
            call(codes, **changed)
    for name in ("starts", "tables", "context"):
        with pytest.raises(TypeError):
            call(c, **{name: dict(zip(names, c.args("cpu")))[name].long()})
    with pytest.raises(TypeError):
        call(codes, ks=codes.k_scales.double())


def test_c_abi_refusals_before_any_launch():
    lib = _lib.load()
    fake, null = ctypes.c_void_p(0x1000), ctypes.c_void_p(0)

    def call(query=fake, k=fake, scales=fake, starts=fake, tables=fake, out=fake, dtype=_lib.CF_BF16,
             form=_lib.CF_CACHE_INT8, pages=100, tokens=16, sequences=4, heads=8, kv_heads=2, dim=64, block=16,
             width=100, ws=fake, ws_bytes=1 << 30):
        return lib.cf_paged_attention_chunk(query, k, fake, scales, fake, starts, tables, fake, out, dtype, form, pages,
                                            tokens, sequences, heads, kv_heads, dim, block, width, 1.0, ws, ws_bytes,
                                            null)

    assert call(tokens=0) == _lib.CF_OK
    for case in ({"query": null}, {"k": null}, {"scales": null}, {"starts": null}, {"tables": null}, {"out": null},
                 {"dtype": 9}, {"form": 9}, {"pages": 0}, {"sequences": -1}, {"kv_heads": 3}, {"kv_heads": 0},
                 {"dim": 1025}, {"block": 0}, {"width": 0}, {"ws": null}, {"ws_bytes": 8},
                 {"ws": ctypes.c_void_p(0x1008)}, {"query": ctypes.c_void_p(0x1001)}, {"pages": 2**27, "block": 16},
                 {"tokens": 2**29}, {"tokens": 2**27, "heads": 8, "width": 1}):
        assert call(**case) == _lib.CF_ERR_INVALID_ARGUMENT, case
    size = lib.cf_paged_attention_chunk_workspace_bytes
    assert size(_lib.CF_BF16, _lib.CF_CACHE_PLAIN, 2048, 1, 32, 8, 128, 16, 128) >= 0
    assert size(_lib.CF_BF16, _lib.CF_CACHE_PLAIN, 16, 1, 8, 3, 64, 16, 10) == 0
