"""Several continuations of shared prompts, sampled on a paged cache: its pages,
the attention over them and the tokens' log probabilities in one run."""

from __future__ import annotations

import torch

import cuda_force_amd as cf
from tests import logprobs_util, shared_util

BLOCK, KV_HEADS, HEADS, DIM, VOCAB, PAGES, ROWS, WIDTH = 16, 2, 8, 64, 611, 40, 9, 8
PROMPTS = (37, 16)  # tokens: a partial last page, and none
CHILDREN = (2, 3, 4, 5, 6, 7)  # rows of the tables: three of each prompt


class Run:
    """The program's state, and beside it what every row holds token by token."""

    def __init__(self, device, dtype):
        gen = torch.Generator().manual_seed(3)

        def normal(*shape, scale=1.0):
            return (scale * torch.randn(*shape, generator=gen)).to(device, dtype)

        self.device, self.dtype = device, dtype
        self.keys, self.values = normal(VOCAB, KV_HEADS, DIM), normal(VOCAB, KV_HEADS, DIM)
        self.queries = normal(VOCAB, HEADS, DIM)
        self.places = normal(WIDTH * BLOCK, 1, DIM, scale=0.3)
        self.head = normal(HEADS * DIM, VOCAB, scale=0.2)
        nothing = torch.full((PAGES, BLOCK, KV_HEADS, DIM), float("nan"), device=device, dtype=dtype)
        self.caches = [nothing, nothing.clone()]
        self.counts = torch.zeros(PAGES, dtype=torch.int32, device=device)
        self.tables = torch.randint(-2**31, 2**31 - 1, (ROWS, WIDTH), generator=gen).to(device, torch.int32)
        self.context = torch.zeros(ROWS, dtype=torch.int32, device=device)
        self.starts = self.ints(0, 3, 6)
        self.prefix = self.ints(*PROMPTS)
        self.tokens = torch.zeros(len(CHILDREN), dtype=torch.int64, device=device)
        self.held: dict[int, list[int]] = {}  # the tokens of every row
        prompts = [torch.randint(0, VOCAB, (n,), generator=gen) for n in PROMPTS]
        for row, prompt in enumerate(prompts):
            slots = cf.cache_extend(self.counts, self.tables, self.context, self.ints(row), BLOCK, len(prompt))[0]
            at = torch.arange(len(prompt), device=device)
            self.write(slots, prompt.to(device), at)
            self.held[row] = prompt.tolist()

    def ints(self, *values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def write(self, slots, tokens, at):
        self.caches[0].view(-1, KV_HEADS, DIM)[slots] = self.keys[tokens] + self.places[at]
        self.caches[1].view(-1, KV_HEADS, DIM)[slots] = self.values[tokens]

    def fork(self, parents, children):
        status = cf.cache_fork(self.caches, self.counts, self.tables, self.context, self.ints(*parents),
                               self.ints(*children))
        assert status.tolist() == [0] * len(parents)
        for p, c in zip(parents, children):
            self.held[c] = list(self.held[p])
            if c in CHILDREN and p in CHILDREN:
                self.tokens[c - CHILDREN[0]] = self.tokens[p - CHILDREN[0]]

    def release(self, *rows):
        cf.cache_release(self.counts, self.tables, self.context, self.ints(*rows), BLOCK)
        for r in rows:
            del self.held[r]

    def compact(self):
        counts, tables, live = cf.cache_compact(self.caches, self.counts, self.tables, self.context)
        n = int(live)
        assert n == int((self.counts > 0).sum()) and (counts[n:] == 0).all() and (counts[:n] > 0).all()
        self.counts.copy_(counts)
        self.tables.copy_(tables)
        for cache in self.caches:
            cache[n:] = float("nan")  # given up

    def step(self):
        """One token for every child, all on the device: nothing is read back."""
        first, last = CHILDREN[0], CHILDREN[-1] + 1
        rows = torch.arange(first, last, dtype=torch.int32, device=self.device)
        at = self.context[first:last].long()
        slots = cf.cache_extend(self.counts, self.tables, self.context, rows, BLOCK)[:, 0]
        self.write(slots, self.tokens, at)
        out = cf.paged_attention_shared(self.queries[self.tokens], *self.caches, self.starts, self.prefix,
                                        self.tables[first:last], self.context[first:last])
        logits = out.view(len(CHILDREN), -1) @ self.head
        got = cf.token_logprobs(logits, self.tokens, scale=0.8, entropy=True, top=3)
        # Child k takes its (k mod 3)-th likeliest token.
        choice = torch.arange(len(CHILDREN), device=self.device) % 3
        following = got.top_tokens.gather(1, choice[:, None])[:, 0]
        return slots, out, logits, got, following

    def check(self, slots, out, logits, got, following):
        """The step's results against every child's own tokens in float64."""
        assert (slots >= 0).all()
        k, v = (c.view(-1, KV_HEADS, DIM).cpu() for c in self.caches)
        tables = self.tables.cpu()
        for i, row in enumerate(CHILDREN):
            self.held[row].append(int(self.tokens[i]))
            tokens = torch.tensor(self.held[row])
            assert int(self.context[row]) == len(tokens)
            at = torch.arange(len(tokens))
            slot = tables[row].long()[at // BLOCK] * BLOCK + at % BLOCK
            assert torch.equal(k[slot], self.keys.cpu()[tokens] + self.places.cpu()[at])
            assert torch.equal(v[slot], self.values.cpu()[tokens])
        case = shared_util.Shared(self.queries[self.tokens].cpu(), *(c.cpu() for c in self.caches), self.starts.cpu(),
                                  self.prefix.cpu(), tables[CHILDREN[0]:CHILDREN[-1] + 1],
                                  self.context.cpu()[CHILDREN[0]:CHILDREN[-1] + 1], DIM ** -0.5)
        shared_util.check(out, case)
        ref = logprobs_util.reference(logits, self.tokens[:, None], 0.8, 3)
        logprobs_util.close(got.logprobs[:, None], ref[0], logprobs_util.logprob_tolerance(ref[0], VOCAB))
        logprobs_util.close(got.entropy, ref[1], logprobs_util.entropy_tolerance(ref[1], VOCAB))
        assert torch.equal(got.top_tokens.cpu(), ref[3])
        self.tokens.copy_(following)


def run(device, dtype, step=None):
    """Prompts, forks, steps, a child replaced by its neighbour's continuation,
    a compaction, and the end. `step`: how a step is made, Run.step by default."""
    r = Run(device, dtype)
    r.fork([0, 0, 0, 1, 1, 1], CHILDREN)
    make = r.step if step is None else step(r)
    for _ in range(14):
        r.check(*make())
    r.release(4)
    r.fork([3], [4])  # rows 3 and 4 share more than their prompt now
    r.tokens[2] = (r.tokens[1] + 1) % VOCAB
    for _ in range(4):
        r.check(*make())
    r.release(0, 7)
    r.fork([6], [7])
    r.compact()
    for _ in range(5):
        r.check(*make())
    r.release(1, *CHILDREN)
    assert (r.counts == 0).all() and (r.context == 0).all()


def step_without_pages(device, make=None):
    """Three sequences take a step of which one finds no free page: its token
    goes to page 0, which no sequence has, and nothing else is touched. `make`:
    how the step is called."""
    pages, block, kv_heads, dim = 6, 4, 2, 8
    gen = torch.Generator().manual_seed(5)
    caches = [torch.randn(pages, block, kv_heads, dim, generator=gen).to(device) for _ in range(2)]
    counts, context = (torch.zeros(n, dtype=torch.int32, device=device) for n in (pages, 3))
    tables = torch.zeros(3, 3, dtype=torch.int32, device=device)
    rows = torch.arange(3, dtype=torch.int32, device=device)
    counts[0] = 1
    for row, length in enumerate((7, 4, 8)):
        assert (cf.cache_extend(counts, tables, context, rows[row : row + 1], block, length) > 0).all()
    assert (counts == 1).all()
    new = torch.randn(3, kv_heads, dim, generator=gen).to(device)

    def step():
        slots = cf.cache_extend(counts, tables, context, rows, block)[:, 0]
        for cache in caches:
            cache.view(-1, kv_heads, dim)[slots.clamp(min=0)] = new
        return slots

    before = [[t.clone() for t in (counts, tables, context)], [c.clone() for c in caches]]
    slots = (step if make is None else make(step, [counts, tables, context, *caches]))()
    own = int(tables[0, 1]) * block + 3
    assert slots.tolist() == [own, -1, -1] and context.tolist() == [8, 4, 8]
    assert torch.equal(counts, before[0][0]) and torch.equal(tables, before[0][1])
    for cache, was in zip(caches, before[1]):
        now, was = cache.view(-1, kv_heads, dim), was.view(-1, kv_heads, dim)
        assert torch.equal(now[own], new[0])
        rest = [i for i in range(block, pages * block) if i != own]
        assert torch.equal(now[rest], was[rest])
