"""Paged caches in the middle of their work."""

from __future__ import annotations

import torch


def state(lengths, block, width, pages, seed=0, tensors=2, shape=(2, 8), dtype=torch.float32):
    """(caches, ref_counts, block_tables, context_lens): rows of the given
    lengths over distinct pages in random order, caches full of numbers, table
    entries behind a length arbitrary."""
    gen = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    tables = torch.randint(-2**31, 2**31 - 1, (len(lengths), width), generator=gen).to(torch.int32)
    counts = torch.zeros(pages, dtype=torch.int32)
    used = 0
    for s, n in enumerate(lengths):
        need = -(-max(n, 0) // block)
        tables[s, :need] = order[used : used + need]
        counts[order[used : used + need].long()] = 1
        used += need
    caches = [(100 * torch.randn(pages, block, *shape, generator=gen)).to(dtype) for _ in range(tensors)]
    return caches, counts, tables, torch.tensor(lengths, dtype=torch.int32)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def to(device, things):
    """A copy on the device, lists inside included."""
    return [to(device, t) if isinstance(t, (list, tuple)) else t.to(device, copy=True) for t in things]


def same(a, b) -> None:
    """Bit for bit."""
    for x, y in zip(a, b, strict=True):
        if isinstance(x, (list, tuple)):
            same(x, y)
        else:
            assert torch.equal(x.cpu().view(torch.uint8) if x.ndim else x.cpu(),
                               y.cpu().view(torch.uint8) if y.ndim else y.cpu())
