"""Calls of the operators of serving in 8 bits that no kernel takes: float64, and
gradients."""

from __future__ import annotations

import pytest
import torch

import cuda_force_amd as cf
from tests import chunk_util, codes_util

pytestmark = pytest.mark.gpu
CODES = [torch.int8, torch.float8_e4m3fn]


@pytest.mark.parametrize("held", CODES)
def test_float64_rows_are_stored_like_others(held, monkeypatch):
    monkeypatch.setenv("CUDAFORGE_STRICT", "0")
    # Multiples of a power of two: many quotients lie in the middle of two codes.
    top = 127 if held == torch.int8 else 448
    steps = torch.arange(-4 * top, 4 * top + 1).double() / 4
    steps = torch.cat([steps, torch.arange(-1024, 1025).double() * 2.0**-11])
    x = torch.stack([steps, steps * 0.0625, steps * 4]).view(3, 1, -1)
    sets = []
    for device in ("cpu", "cuda"):
        k, v = (torch.zeros(1, 4, 1, x.shape[-1], device=device).to(held) for _ in range(2))
        s, t = (torch.zeros(1, 4, 1, device=device) for _ in range(2))
        ones = torch.arange(3, device=device)
        if device == "cuda":
            with pytest.warns(RuntimeWarning):
                cf.cache_write(x.to(device), -x.to(device), k, v, ones, s, t)
        else:
            cf.cache_write(x, -x, k, v, ones, s, t)
        sets.append([a.float().cpu() for a in (k, v, s, t)])
    numbers, scales = codes_util.rows(x, held)
    assert torch.equal(sets[0][0].view(4, -1)[:3].double(), numbers.view(3, -1))
    for a, b in zip(*sets):
        assert torch.equal(a, b)


@pytest.mark.parametrize("held", [None, *CODES])
def test_gradients_of_chunks(held):
    """Of the query, and of plain caches: as on the CPU."""
    c = chunk_util.build([(5, 40), (1, 33), (0, 7), (9, 9)], 4, 2, 32, 16, torch.float32, held, behind=2, bad=False)
    grads = []
    for device in ("cpu", "cuda"):
        args = [t if t is None or isinstance(t, float) else t.clone() for t in c.args(device)]
        leaves = [args[0], *(args[1:3] if held is None else [])]
        for t in leaves:
            t.requires_grad_(True)
        out = cf.paged_attention_chunk(*args)
        (out * torch.linspace(-1, 1, out.numel(), device=device).view(out.shape)).sum().backward()
        grads.append([t.grad.cpu() for t in leaves])
    for a, b in zip(*grads):
        assert torch.isfinite(b).all() and a.abs().max() > 0
        assert (a - b).abs().max() <= 2.0**-16 * a.abs().max()
