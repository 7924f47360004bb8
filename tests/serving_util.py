"""A decoder layer's attention served in 8 bits: int8 projections, a paged cache
of codes, chunks and single tokens."""

from __future__ import annotations

import math

import torch

import cuda_force_amd as cf
from tests import chunk_util


def code_rows(x, held):
    """(numbers of the codes, scales) of the rows, by their definition. The
    quotient of two fp32 numbers is a tie or at least 2^-49 from one, so rounding
    it to fp64 first moves none."""
    x = x.detach().cpu().float()
    top = 127.0 if held == torch.int8 else 448.0
    scales = x.abs().amax(-1) * (torch.tensor(1.0) / top)
    scales = torch.where(scales > 0, scales, 1.0)
    q = x.double() / scales.double()[..., None]
    if held == torch.int8:
        return q.round(), scales
    step = torch.exp2(torch.frexp(q)[1].clamp(min=-5).double() - 4)  # four bits, from 2^-6 on
    return (q / step).round() * step, scales


class Layer:
    HEADS, KV_HEADS, DIM, BLOCK, PAGES, ROWS = 8, 2, 64, 16, 40, 4

    def __init__(self, device, dtype, held, seed=0):
        self.device, self.dtype, self.held = device, dtype, held
        gen = torch.Generator().manual_seed(seed)
        self.hidden = self.HEADS * self.DIM
        out = (self.HEADS + 2 * self.KV_HEADS) * self.DIM

        def weight(n, k):
            w = torch.randn(n, k, generator=gen) / math.sqrt(k)
            return cf.quantize_int8_rows(w.to(device))

        self.into, self.into_scales = weight(out, self.hidden)
        self.back, self.back_scales = weight(self.hidden, self.hidden)
        shape = (self.PAGES, self.BLOCK, self.KV_HEADS)
        self.caches = [torch.zeros(*shape, self.DIM, dtype=held or dtype, device=device) for _ in range(2)]
        self.scales = [torch.zeros(shape, device=device) if held else None for _ in range(2)]
        self.counts = torch.zeros(self.PAGES, dtype=torch.int32, device=device)
        self.tables = torch.zeros(self.ROWS, self.PAGES // 2, dtype=torch.int32, device=device)
        self.lens = torch.zeros(self.ROWS, dtype=torch.int32, device=device)
        self.gen = gen

    def ints(self, *values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def tokens(self, n):
        return torch.randn(n, self.hidden, generator=self.gen).to(self.dtype).to(self.device)

    def linear(self, x, weight, scales):
        codes, of_rows = cf.quantize_int8_rows(x)
        return cf.matmul_int8(codes, weight, of_rows, scales, dtype=self.dtype)

    def project(self, x):
        """Views of the fused projection: query, keys, values."""
        y = self.linear(x, self.into, self.into_scales).view(x.shape[0], -1, self.DIM)
        return y.split([self.HEADS, self.KV_HEADS, self.KV_HEADS], 1)

    def step(self, x, slots, starts):
        """New tokens x at `slots` (their places), sequence by sequence."""
        q, k, v = self.project(x)
        cf.cache_write(k, v, *self.caches, slots, *self.scales)
        out = cf.paged_attention_chunk(q, *self.caches, starts, self.tables, self.lens, *self.scales)
        return out, self.linear(out.flatten(1), self.back, self.back_scales)

    def extend(self, sequences, tokens):
        """Slots of `tokens` new tokens of each of the rows, in their order."""
        got = [cf.cache_extend(self.counts, self.tables, self.lens, self.ints(s), self.BLOCK, tokens)
               for s in sequences]
        slots = torch.cat(got).view(-1)
        assert (slots >= 0).all()
        return slots

    def starts(self, new):
        return self.ints(0, *torch.tensor([new.get(s, 0) for s in range(self.ROWS)]).cumsum(0).tolist())

    def fork(self, parent, child):
        done = cf.cache_fork(self.caches, self.counts, self.tables, self.lens, self.ints(parent), self.ints(child))
        assert done.tolist() == [0]
        if self.held:
            # The last page is the child's own if it is not full; its scales follow the codes.
            last = (self.lens[parent].long() - 1) // self.BLOCK
            cf.cache_copy(self.scales, self.tables[parent, last].view(1), self.tables[child, last].view(1))

    def compact(self):
        """Pages in use to the front, scales along with the codes."""
        if self.held:
            cf.cache_compact(self.scales, self.counts, self.tables, self.lens)
        self.counts, self.tables, _ = cf.cache_compact(self.caches, self.counts, self.tables, self.lens)

    # ---- what a step has to give ------------------------------------------------

    def check_linear(self, x, weight, scales, got):
        """The product of the codes is exact; each of the three fp32 steps and the
        result's rounding is off by half a step (of fp16 at least 2^-24, its step
        below 2^-14: 2^-25 is more than 2^-11 of such a result)."""
        numbers, of_rows = code_rows(x, torch.int8)
        exact = numbers @ weight.cpu().double().T
        want = exact * of_rows.double()[:, None] * scales.cpu().double()
        half = torch.finfo(self.dtype).eps / 2
        least = 2.0**-25 if self.dtype == torch.float16 else 0.0
        assert ((got.cpu().double() - want).abs() <= (half * 1.01 + 3 * 2.0**-24) * want.abs() + least).all()

    def check_step(self, x, slots, starts, out, y):
        q, k, v = self.project(x)
        self.check_linear(x, self.into, self.into_scales, torch.cat([q, k, v], 1).flatten(1))
        back = cf.cache_read(*self.caches, slots, *self.scales, dtype=self.dtype)
        for given, kept in zip((k, v), back):
            if self.held:
                numbers, scales = code_rows(given, self.held)
                want = (numbers.float() * scales[..., None]).to(self.dtype)
            else:
                want = given.cpu()
            assert torch.equal(kept.cpu(), want)
        cpu = [None if t is None else t.cpu() for t in (q, *self.caches, starts, self.tables, self.lens, *self.scales)]
        chunk_util.check(out, chunk_util.Chunks(*cpu, 1.0 / math.sqrt(self.DIM)))
        self.check_linear(out.flatten(1), self.back, self.back_scales, y)

    def run(self, new):
        """`new`: tokens of each row that gets some, as {row: count}."""
        slots = torch.cat([self.extend([s], n) for s, n in sorted(new.items())])
        starts = self.starts(new)
        x = self.tokens(len(slots))
        out, y = self.step(x, slots, starts)
        self.check_step(x, slots, starts, out, y)
        return out, y


def serve(layer: Layer) -> None:
    """Prompts whole and in chunks, single tokens, forks, a release, pages moved."""
    layer.run({0: 37, 1: 16})
    layer.run({0: 1, 1: 1, 2: 5})
    layer.run({2: 40, 0: 1})  # a chunk's end and a single token in one batch
    layer.fork(0, 3)
    layer.run({0: 1, 3: 1})
    layer.run({0: 3, 1: 1, 2: 1, 3: 18})
    cf.cache_release(layer.counts, layer.tables, layer.lens, layer.ints(1), layer.BLOCK)
    layer.compact()
    layer.run({0: 1, 2: 1, 3: 1})
    layer.run({1: 20, 2: 1})
