"""Paged caches with shared prompts, and attention over them in float64."""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch


@dataclass
class Shared:
    query: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    starts: torch.Tensor
    prefix: torch.Tensor
    tables: torch.Tensor
    context: torch.Tensor
    scale: float

    def args(self, device="cuda"):
        return [t.to(device) for t in (self.query, self.k, self.v, self.starts, self.prefix, self.tables,
                                       self.context)] + [self.scale]


def build(groups, heads, kv_heads, dim, block, dtype, seed=0, loners=0, spare=3, fill=float("nan"), copies=False):
    """`groups`: (prefix length, context lengths of its sequences) each; `loners`
    sequences of 5, 10, ... tokens follow that no group holds. Whole prefix
    pages are shared (copies: every sequence has its own), the partial one is
    copied. Everything no token lies in holds `fill`; pages are dealt in random
    order."""
    gen = torch.Generator().manual_seed(seed)
    starts, lengths, prefix = [0], [], []
    for p, contexts in groups:
        prefix.append(p)
        lengths += contexts
        starts.append(len(lengths))
    lengths += [5 * (i + 1) for i in range(loners)]
    width = max([1] + [-(-n // block) for n in lengths])
    total = spare + sum(-(-n // block) for n in lengths) + sum(-(-p // block) for p in prefix)
    order = torch.randperm(total, generator=gen).tolist()
    k = torch.full((total, block, kv_heads, dim), fill)
    v = k.clone()
    tables = torch.randint(-2**31, 2**31 - 1, (len(lengths), width), generator=gen).to(torch.int32)
    s = 0

    def store(page, at, kk, vv):
        k[page, at : at + len(kk)] = kk
        v[page, at : at + len(vv)] = vv

    def normal(n):
        return torch.randn(n, kv_heads, dim, generator=gen)

    for p, contexts in [*groups, *[(0, [n]) for n in lengths[starts[-1]:]]]:
        pk, pv = normal(p), normal(p)
        pages = [] if copies else [order.pop() for _ in range(p // block)]
        for i, page in enumerate(pages):
            store(page, 0, pk[i * block : (i + 1) * block], pv[i * block : (i + 1) * block])
        for n in contexts:
            kk = torch.cat([pk, normal(max(n - p, 0))])[:n]
            vv = torch.cat([pv, normal(max(n - p, 0))])[:n]
            for i in range(-(-n // block)):
                if i < len(pages) and (i + 1) * block <= n:
                    tables[s, i] = pages[i]
                    continue
                page = order.pop()
                store(page, 0, kk[i * block : (i + 1) * block], vv[i * block : (i + 1) * block])
                tables[s, i] = page
            s += 1
    query = torch.randn(len(lengths), heads, dim, generator=gen)
    return Shared(query.to(dtype), k.to(dtype), v.to(dtype), torch.tensor(starts, dtype=torch.int32),
                  torch.tensor(prefix, dtype=torch.int32), tables, torch.tensor(lengths, dtype=torch.int32),
                  1.0 / math.sqrt(dim))


def reference(c: Shared):
    """(out, sum of p |v|) in float64, sequence by sequence."""
    pages, block, kv_heads, dim = c.k.shape
    heads = c.query.shape[1]
    out = torch.zeros(c.query.shape, dtype=torch.float64)
    size = torch.zeros_like(out)
    for s, n in enumerate(c.context.tolist()):
        t = torch.arange(min(max(n, 0), c.tables.shape[1] * block))
        page = c.tables[s].long()[t // block]
        there = (page >= 0) & (page < pages)
        slot = (page * block + t % block)[there]
        if slot.numel() == 0:
            continue
        k = c.k.view(-1, kv_heads, dim)[slot].double().permute(1, 2, 0)
        v = c.v.view(-1, kv_heads, dim)[slot].double().permute(1, 0, 2)
        q = c.query[s].double().view(kv_heads, -1, dim)
        p = torch.softmax(q @ k * c.scale, -1)
        out[s] = (p @ v).view(heads, dim)
        size[s] = (p @ v.abs()).view(heads, dim)
    return out, size


def check(got: torch.Tensor, c: Shared) -> None:
    """Within the roundings: the result to its type, the probabilities to the
    cache's (half an ulp each: relative to sum p |v|), and fp32 scores and sums
    (an exponent of up to about 2^6 with 128 to 256 roundings of 2^-24 of its
    terms, a chain of tokens / 32 accumulations)."""
    ref, size = reference(c)
    half = torch.finfo(c.query.dtype).eps / 2
    f32 = 2.0**-16 + 2.0**-24 * float(c.context.max()) / 32
    tolerance = (f32 + (half if c.query.dtype != torch.float32 else 0.0)) * size + half * ref.abs()
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    worst = ((got - ref).abs() - tolerance).max().item()
    assert worst <= 0, worst
