"""Batches of chunks over paged caches, and attention of them in float64."""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

CODES = [torch.int8, torch.float8_e4m3fn]


@dataclass
class Chunks:
    query: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    starts: torch.Tensor
    tables: torch.Tensor
    context: torch.Tensor
    k_scales: torch.Tensor | None
    v_scales: torch.Tensor | None
    scale: float

    def args(self, device="cuda"):
        return [None if t is None else t.to(device) for t in (
            self.query, self.k, self.v, self.starts, self.tables, self.context, self.k_scales, self.v_scales)
        ] + [self.scale]


def build(sequences, heads, kv_heads, dim, block, dtype, held=None, seed=0, before=0, behind=0, spare=3, bad=True):
    """`sequences`: (new tokens, context) each; `before` and `behind` rows that no
    sequence holds. `held`: the type of an 8-bit cache. Where no token lies the
    cache holds NaN (codes of NaN, or any with NaN scales), unless not `bad`;
    pages are dealt in random order."""
    gen = torch.Generator().manual_seed(seed)
    starts = [before]
    for n, _ in sequences:
        starts.append(starts[-1] + n)
    lengths = [c for _, c in sequences]
    width = max([1] + [-(-c // block) for c in lengths])
    total = spare + sum(-(-c // block) for c in lengths)
    order = torch.randperm(total, generator=gen).tolist()
    tables = torch.randint(-2**31, 2**31 - 1, (len(lengths), width), generator=gen).to(torch.int32)
    used = torch.zeros(total, block, dtype=torch.bool)
    for s, c in enumerate(lengths):
        for i in range(-(-c // block)):
            tables[s, i] = order.pop()
            used[tables[s, i], : min(block, c - i * block)] = True
    caches, scales = [], []
    for _ in range(2):
        x = torch.randn(total, block, kv_heads, dim, generator=gen)
        if held is None:
            if bad:
                x[~used] = float("nan")
            caches.append(x.to(dtype))
            scales.append(None)
            continue
        top = 127.0 if held == torch.int8 else 448.0
        # Any scales, not those of these codes alone: sizes differ from token to token.
        s = torch.exp(torch.randn(total, block, kv_heads, generator=gen)) / top
        codes = (x / x.abs().amax(-1, keepdim=True) * top).clamp(-top, top)
        codes = codes.round() if held == torch.int8 else codes
        codes = codes.to(held)
        if bad:
            s[~used] = float("nan")
            if held != torch.int8:
                codes.view(torch.uint8)[~used] = 0x7F
        caches.append(codes)
        scales.append(s)
    query = torch.randn(starts[-1] + behind, heads, dim, generator=gen)
    return Chunks(query.to(dtype), caches[0], caches[1], torch.tensor(starts, dtype=torch.int32), tables,
                  torch.tensor(lengths, dtype=torch.int32), scales[0], scales[1], 1.0 / math.sqrt(dim))


def reference(c: Chunks):
    """(out, sum of p |v|) in float64, row by row."""
    pages, block, kv_heads, dim = c.k.shape
    tokens, heads = c.query.shape[:2]
    out = torch.zeros(c.query.shape, dtype=torch.float64)
    size = torch.zeros_like(out)
    done = 0
    for s, length in enumerate(c.context.tolist()):
        first = max(done, min(max(int(c.starts[s]), 0), tokens))
        end = max(first, min(max(int(c.starts[s + 1]), 0), tokens))
        done = end
        if first == end:
            continue
        length = min(max(length, 0), c.tables.shape[1] * block)
        t = torch.arange(length)
        page = c.tables[s].long()[t // block]
        there = (page >= 0) & (page < pages)
        at = (page * block + t % block)[there]

        def rows(cache, scales):
            x = cache.float().view(-1, kv_heads, dim)[at].double()
            return x if scales is None else x * scales.view(-1, kv_heads)[at].double()[..., None]

        k, v = rows(c.k, c.k_scales), rows(c.v, c.v_scales)
        for i in range(end - first):
            n = int((t[there] <= length - (end - first) + i).sum())
            if n == 0:
                continue
            q = c.query[first + i].double().view(kv_heads, -1, dim)
            p = torch.softmax(q @ k[:n].permute(1, 2, 0) * c.scale, -1)
            out[first + i] = (p @ v[:n].permute(1, 0, 2)).view(heads, dim)
            size[first + i] = (p @ v[:n].abs().permute(1, 0, 2)).view(heads, dim)
    return out, size


def check(got: torch.Tensor, c: Chunks) -> None:
    """Within the roundings: the result to its type, the weights to the tiles'
    (the query's type; fp16 for codes, where an fp32 query's are the sum of two
    fp16 numbers), half an ulp each relative to sum p |v|, and fp32 scores and
    sums (an exponent of up to about 2^6 with 128 to 256 roundings of 2^-24 of
    its terms, or an fp32 query's 2^-22 beside codes; a chain of tokens / 32
    accumulations). fp16 weights are off by at most 2^-38 of a row's largest
    below 2^-27 of it."""
    ref, size = reference(c)
    half = torch.finfo(c.query.dtype).eps / 2
    codes = c.k_scales is not None
    longest = float(max(c.context.max(), 1))
    tolerance = (2.0**-16 + 2.0**-24 * longest / 32) * size + half * ref.abs()
    if c.query.dtype != torch.float32:
        tolerance += (2.0**-11 if codes else half) * size
    if codes or c.query.dtype == torch.float16:
        v = c.v.float().nan_to_num(0.0, 0.0, 0.0).abs()
        if codes:
            v = v * c.v_scales.nan_to_num(0.0, 0.0, 0.0).abs()[..., None]
        tolerance += 2.0**-37 * longest * float(v.max())
    if c.query.dtype == torch.float16:
        # Below 2^-14 fp16 has steps of 2^-24 whatever the value: half of one is
        # more than 2^-11 of such a result (3.0e-8 against 4.4e-9 at 9e-6).
        tolerance += 2.0**-25
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    worst = ((got - ref).abs() - tolerance).max().item() if got.numel() else 0.0
    assert worst <= 0, worst
