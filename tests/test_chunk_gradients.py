"""Gradients of attention of chunks through the PyTorch composition, against
differences in float64."""

from __future__ import annotations

import pytest
import torch

import cuda_force_amd as cf
from tests import chunk_util


@pytest.mark.parametrize("bad", [False, True])
def test_gradients_of_query_and_caches(bad):
    """Rows before, behind and of no sequence, more rows than context, pages left
    out; places of no token hold NaN."""
    c = chunk_util.build([(3, 10), (1, 6), (0, 4), (4, 2)], 4, 2, 4, 4, torch.float64, before=1, behind=1, bad=bad)
    c.tables[0, 0] = -1
    leaves = [t.clone().requires_grad_(True) for t in (c.query, c.k, c.v)]

    def attend(q, k, v):
        return cf.paged_attention_chunk(q, k, v, c.starts, c.tables, c.context, scale=c.scale)

    weight = torch.randn(c.query.shape, dtype=torch.float64)
    grads = torch.autograd.grad((attend(*leaves) * weight).sum(), leaves)
    gen = torch.Generator().manual_seed(1)
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        assert torch.isfinite(grad).all() and grad.abs().max() > 0
        step = torch.randn(leaf.shape, generator=gen, dtype=torch.float64) * 1e-5
        values = []
        for sign in (1, -1):
            moved = [t.detach().clone() for t in leaves]
            moved[i] = moved[i] + sign * step
            values.append((attend(*moved) * weight).sum())
        # The third derivative's share is about step^2 of it, the fp64 sums' 2^-52 over the step.
        assert abs((values[0] - values[1]) / 2 - (grad * step).sum()) <= 1e-8 * (grad.abs() * step.abs()).sum()


def test_a_cache_alone_may_need_a_gradient():
    c = chunk_util.build([(3, 10)], 2, 1, 8, 4, torch.float32)
    v = c.v.clone().requires_grad_(True)
    out = cf.paged_attention_chunk(c.query, c.k, v, c.starts, c.tables, c.context)
    out.sum().backward()
    # Weights of a row sum to 1.
    assert abs(v.grad.sum().item() - out.numel()) <= 1e-4 * out.numel()
