"""The operators of generation from a shared prompt, as measurable cases.

Each case is a plain dict: ``kind`` names the operator, the rest its sizes.
``run`` with ``own`` false computes it from elementary torch operations, with
``own`` true through the package's entry points.

Kinds:

* ``attention`` one decode step over a paged cache whose sequences share long
                prompts in groups;
* ``logprobs``  log probabilities of given tokens, entropy and the likeliest
                alternatives, from a step's logits;
* ``likelihood`` the same as a training loss: log probabilities and entropy
                forward, the gradient of the logits backward;
* ``fork``      candidates forked from running sequences, grown by a token and
                dropped again;
* ``copy``      whole pages copied inside a cache;
* ``compact``   the live pages of a fragmented cache moved to its front.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed() -> list[dict]:
    return [
        # Eight answers being sampled for one question: the latency case.
        {"name": "attention_few", "kind": "attention", "dtype": "bf16", "sequences": 8, "groups": 1, "prefix": 1000,
         "suffix": 60, "heads": 32, "kv_heads": 8, "dim": 128, "block": 16},
        # A chat server's batch behind one system prompt.
        {"name": "attention_batch", "kind": "attention", "dtype": "bf16", "sequences": 64, "groups": 1,
         "prefix": 4099, "suffix": 500, "heads": 32, "kv_heads": 8, "dim": 128, "block": 16},
        # Many questions about one long document: the largest.
        {"name": "attention_document", "kind": "attention", "dtype": "bf16", "sequences": 128, "groups": 1,
         "prefix": 32768, "suffix": 256, "heads": 32, "kv_heads": 8, "dim": 128, "block": 32},
        # Several prompts, some samples of each, every query head with its own keys.
        {"name": "attention_groups", "kind": "attention", "dtype": "f16", "sequences": 37, "groups": 5, "prefix": 2001,
         "suffix": 333, "heads": 16, "kv_heads": 16, "dim": 64, "block": 16},
        # The same step in full precision.
        {"name": "attention_f32", "kind": "attention", "dtype": "f32", "sequences": 16, "groups": 2, "prefix": 2048,
         "suffix": 200, "heads": 32, "kv_heads": 8, "dim": 128, "block": 16},
        # What a sampler reports with each generated token.
        {"name": "logprobs_step", "kind": "logprobs", "dtype": "bf16", "rows": 8, "vocab": 50257, "count": 1,
         "top": 20, "entropy": True, "scale": 1.25},
        # Scoring four answers at each position of a prompt, from full-precision logits in a padded buffer.
        {"name": "logprobs_score", "kind": "logprobs", "dtype": "f32", "rows": 1001, "vocab": 32000, "count": 4,
         "top": 0, "entropy": False, "scale": 1.0},
        # A large vocabulary with its five likeliest tokens at every position.
        {"name": "logprobs_wide", "kind": "logprobs", "dtype": "f16", "rows": 600, "vocab": 131072, "count": 1,
         "top": 5, "entropy": True, "scale": 0.7},
        # A policy-gradient step with an entropy bonus, padded positions among its tokens.
        {"name": "likelihood_train", "kind": "likelihood", "dtype": "bf16", "rows": 4096, "vocab": 32000, "count": 1,
         "entropy": True, "scale": 1.0},
        # A step of search: four candidates of each of eight sequences.
        {"name": "fork_step", "kind": "fork", "parents": 8, "each": 4, "context": 1000, "block": 16, "heads": 8,
         "dim": 128, "layers": 4, "dtype": "bf16"},
        # Pages of a finished prompt copied to a place of their own.
        {"name": "copy_pages", "kind": "copy", "pages": 4096, "pairs": 1500, "block": 16, "heads": 8, "dim": 128,
         "layers": 2, "dtype": "bf16"},
        # A cache left with holes by finished sequences.
        {"name": "compact_cache", "kind": "compact", "sequences": 48, "context": 1500, "block": 16, "heads": 8,
         "dim": 64, "layers": 2, "dtype": "bf16"},
    ]


def _log(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    kind = rng.choice(["attention"] * 5 + ["logprobs"] * 3 + ["likelihood"] * 2 + ["fork", "copy", "compact"])
    if kind == "attention":
        heads, kv_heads = rng.choice([(32, 8), (32, 32), (16, 16), (32, 4), (24, 8), (64, 8)])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        sequences = _log(rng, 1, 128)
        return {"kind": kind, "dtype": dtype, "sequences": sequences, "groups": rng.randint(1, min(6, sequences)),
                "prefix": _log(rng, 16, 4096 if dtype == "f32" or kv_heads > 8 else 8192), "suffix": _log(rng, 1, 600),
                "heads": heads, "kv_heads": kv_heads, "dim": rng.choice([64, 128, 128]),
                "block": rng.choice([16, 16, 32, 64])}
    if kind == "logprobs":
        vocab = rng.choice([32000, 50257, 65536, 131072, _log(rng, 500, 131072)])
        return {"kind": kind, "dtype": rng.choice(["bf16", "f16", "f32"]), "rows": _log(rng, 1, 600), "vocab": vocab,
                "count": rng.choice([1, 1, 1, 3, 8]), "top": rng.choice([0, 1, 5, 20, 32]),
                "entropy": rng.random() < 0.5, "scale": rng.choice([1.0, 0.7, 1.25])}
    if kind == "likelihood":
        return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "rows": _log(rng, 8, 1500),
                "vocab": rng.choice([32000, 50257, 32001, _log(rng, 1000, 65536)]), "count": rng.choice([1, 1, 5]),
                "entropy": rng.random() < 0.5, "scale": rng.choice([1.0, 0.8])}
    if kind == "fork":
        return {"kind": kind, "parents": _log(rng, 1, 32), "each": rng.randint(1, 6), "context": _log(rng, 2, 2500),
                "block": rng.choice([16, 32]), "heads": rng.choice([8, 16]), "dim": rng.choice([64, 128]),
                "layers": rng.randint(1, 4), "dtype": rng.choice(["bf16", "f32"])}
    if kind == "copy":
        pages = _log(rng, 64, 4096)
        return {"kind": kind, "pages": pages, "pairs": max(1, int(pages * rng.uniform(0.05, 0.4))),
                "block": rng.choice([16, 32]), "heads": 8, "dim": rng.choice([64, 128]), "layers": rng.randint(1, 2),
                "dtype": "bf16"}
    return {"kind": kind, "sequences": _log(rng, 2, 64), "context": _log(rng, 20, 1200), "block": rng.choice([16, 32]),
            "heads": 8, "dim": rng.choice([64, 128]), "layers": rng.randint(1, 2), "dtype": rng.choice(["bf16", "f32"])}


# ---------------------------------------------------------------------------
# Sizes that follow from a case alone.
# ---------------------------------------------------------------------------


def _groups(case: dict) -> tuple[list[int], list[int], list[int], list[int]]:
    """(first sequence of each group and the end, prompt lengths, group of
    each sequence, context lengths): uneven groups, ragged lengths."""
    s, g = case["sequences"], case["groups"]
    starts = [i * s // g for i in range(g + 1)]
    prefix = [case["prefix"] - (i * 131) % (case["prefix"] // 4 + 1) for i in range(g)]
    member = [next(i for i in range(g) if starts[i] <= k < starts[i + 1]) for k in range(s)]
    suffix = [1 + (k * 7919 + case["suffix"] - 1) % case["suffix"] for k in range(s)]
    return starts, prefix, member, [prefix[m] + n for m, n in zip(member, suffix)]


def _lengths(count: int, longest: int) -> list[int]:
    low = max(1, longest // 3)
    return [longest - (i * 7919) % (longest - low + 1) for i in range(count)]


# ---------------------------------------------------------------------------
# Inputs.
# ---------------------------------------------------------------------------


class _Inputs:
    """Seeded values on the GPU."""

    def __init__(self, seed: int) -> None:
        self.gen = torch.Generator(device="cuda").manual_seed(1_000_003 * (seed % 1_000_003) + 29)

    def normal(self, *shape: int, std: float = 1.0, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return torch.randn(*shape, generator=self.gen, device="cuda").mul_(std).to(dtype)

    def whole(self, low: int, high: int, *shape: int) -> torch.Tensor:
        return torch.randint(low, high, shape, generator=self.gen, device="cuda")

    def order(self, count: int) -> torch.Tensor:
        return torch.randperm(count, generator=self.gen, device="cuda")


def _i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case: dict, seed: int) -> dict:
    return _PREPARE[case["kind"]](case, _Inputs(seed))


def _prepare_attention(case: dict, inputs: _Inputs) -> dict:
    dtype = _DTYPES[case["dtype"]]
    s, bs, kvh, d = case["sequences"], case["block"], case["kv_heads"], case["dim"]
    starts, prefix, member, context = _groups(case)
    width = max((c + bs - 1) // bs for c in context)
    shared = [p // bs for p in prefix]  # whole pages of each prompt
    own_pages = [(c + bs - 1) // bs - shared[m] for c, m in zip(context, member)]
    total = sum(shared) + sum(own_pages)
    order = inputs.order(total).to(torch.int32).cpu()
    tables = torch.zeros(s, width, dtype=torch.int32)
    used, prompt = 0, []
    for n in shared:
        prompt.append(order[used:used + n])
        used += n
    for k in range(s):
        n = shared[member[k]]
        tables[k, :n] = prompt[member[k]]
        tables[k, n:n + own_pages[k]] = order[used:used + own_pages[k]]
        used += own_pages[k]
    tables = tables.cuda()
    caches = [inputs.normal(total, bs, kvh, d, dtype=dtype) for _ in range(2)]
    # The part of a prompt behind its last whole page: every sequence holds a copy.
    for m, p in enumerate(prefix):
        if p % bs:
            pages = tables[starts[m]:starts[m + 1], shared[m]].long()
            for cache in caches:
                cache[pages, :p % bs] = cache[pages[0], :p % bs]
    return {"kind": "attention", "q": inputs.normal(s, case["heads"], d, dtype=dtype), "k": caches[0], "v": caches[1],
            "starts": _i32(starts), "prefix": _i32(prefix), "tables": tables, "context": _i32(context),
            "scale": 1.0 / math.sqrt(d), "largest": max(b - a for a, b in zip(starts, starts[1:])),
            "longest": max(prefix), "tail": max(c - prefix[m] for c, m in zip(context, member))}


def _prepare_logits(case: dict, inputs: _Inputs) -> dict:
    rows, vocab, count = case["rows"], case["vocab"], case["count"]
    # Logits as a model gives them: a bulk, a few likely tokens above it, in
    # rows padded to a multiple of 64; every seventh row under a mask.
    pitch = (vocab + 63) // 64 * 64
    wide = inputs.normal(rows, pitch, std=2.0)
    peaks = inputs.whole(0, vocab, rows, 8)
    wide.scatter_add_(1, peaks, inputs.normal(rows, 8, std=3.0).abs_() + 4.0)
    if case["kind"] == "logprobs":
        wide[::7, vocab // 3:vocab // 2] = float("-inf")
    tokens = inputs.whole(0, vocab // 3, rows, count)
    tokens[:, 0] = torch.where(inputs.whole(0, 2, rows) > 0, peaks[:, 0] % (vocab // 3), tokens[:, 0])
    state = {"kind": case["kind"], "logits": wide.to(_DTYPES[case["dtype"]])[:, :vocab], "scale": case["scale"],
             "entropy": case["entropy"], "top": case.get("top", 0)}
    if case["kind"] == "likelihood":
        tokens[::11] = -100  # padding
        state["grad_logprobs"] = inputs.normal(rows, count, std=1.0 / rows)
        state["grad_entropy"] = inputs.normal(rows, std=0.01 / rows)
        if count == 1:
            state["grad_logprobs"] = state["grad_logprobs"][:, 0].contiguous()
        state["logits"].requires_grad_(True)
    state["tokens"] = tokens[:, 0].contiguous() if count == 1 else tokens
    return state


def _caches(case: dict, inputs: _Inputs, pages: int) -> list[torch.Tensor]:
    return [inputs.normal(pages, case["block"], case["heads"], case["dim"], dtype=_DTYPES[case["dtype"]])
            for _ in range(2 * case["layers"])]


def _fork_pages(case: dict) -> tuple[int, int]:
    """(table width, pages of the pool): a third of it free."""
    width = (case["context"] + 1 + case["block"] - 1) // case["block"] + 1
    used = sum((c + case["block"] - 1) // case["block"] for c in _lengths(case["parents"], case["context"]))
    return width, (used + 2 * case["parents"] * case["each"]) * 3 // 2


def _prepare_fork(case: dict, inputs: _Inputs) -> dict:
    bs, n = case["block"], case["parents"]
    children = n * case["each"]
    width, pages = _fork_pages(case)
    lengths = _lengths(n, case["context"])
    order = inputs.order(pages).to(torch.int32).cpu()
    tables = torch.zeros(n + children, width, dtype=torch.int32)
    counts = torch.zeros(pages, dtype=torch.int32)
    used = 0
    for k, length in enumerate(lengths):
        need = (length + bs - 1) // bs
        tables[k, :need] = order[used:used + need]
        used += need
    counts[order[:used].long()] = 1
    parents = [k for k in range(n) for _ in range(case["each"])]
    return {"kind": "fork", "caches": _caches(case, inputs, pages), "counts": counts.cuda(), "tables": tables.cuda(),
            "context": _i32(lengths + [0] * children), "parents": _i32(parents),
            "children": (n + inputs.order(children)).to(torch.int32), "block": bs}


def _prepare_copy(case: dict, inputs: _Inputs) -> dict:
    order = inputs.order(case["pages"]).to(torch.int32)
    n = case["pairs"]
    return {"kind": "copy", "caches": _caches(case, inputs, case["pages"]), "src": order[:n].contiguous(),
            "dst": order[n:2 * n].contiguous()}


def _prepare_compact(case: dict, inputs: _Inputs) -> dict:
    bs = case["block"]
    lengths = _lengths(case["sequences"], case["context"])
    needs = [(c + bs - 1) // bs for c in lengths]
    pages = 2 * sum(needs)
    order = inputs.order(pages).to(torch.int32).cpu()
    tables = torch.zeros(case["sequences"], max(needs), dtype=torch.int32)
    counts = torch.zeros(pages, dtype=torch.int32)
    used = 0
    for k, need in enumerate(needs):
        tables[k, :need] = order[used:used + need]
        if k % 4 == 1:  # the first half is the sequence before's
            half = min(need, needs[k - 1]) // 2
            tables[k, :half] = tables[k - 1, :half]
        used += need
        counts.index_add_(0, tables[k, :need].long(), torch.ones(need, dtype=torch.int32))
    return {"kind": "compact", "caches": _caches(case, inputs, pages), "counts": counts.cuda(),
            "tables": tables.cuda(), "context": _i32(lengths)}


_PREPARE = {"attention": _prepare_attention, "logprobs": _prepare_logits, "likelihood": _prepare_logits,
            "fork": _prepare_fork, "copy": _prepare_copy, "compact": _prepare_compact}


# ---------------------------------------------------------------------------
# One pass.
# ---------------------------------------------------------------------------


def run(state: dict):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


def _own_attention(st: dict):
    import cuda_force_amd as cf

    return cf.paged_attention_shared(st["q"], st["k"], st["v"], st["starts"], st["prefix"], st["tables"],
                                     st["context"], st["scale"])


def _plain_attention(st: dict):
    q, starts, prefix, context = st["q"].float(), st["starts"].long(), st["prefix"].long(), st["context"].long()
    tables = st["tables"].long()
    s, heads, d = q.shape
    pages, bs, kvh, _ = st["k"].shape
    per = heads // kvh
    device = q.device
    groups = prefix.numel()
    # Prompts: each group's rows against one gather of its keys.
    place = starts[:-1, None] + torch.arange(st["largest"], device=device)  # [G, N]
    present = place < starts[1:, None]
    place = torch.where(present, place, starts[:-1, None])
    t = torch.arange(st["longest"], device=device)
    slot = tables[starts[:-1]][:, t // bs] * bs + t % bs  # [G, Lp]
    keys = st["k"].view(pages * bs, kvh, d)[slot].float().permute(0, 2, 3, 1).contiguous()  # [G, KVH, D, Lp]
    values = st["v"].view(pages * bs, kvh, d)[slot].float().permute(0, 2, 1, 3).contiguous()
    rows = q.view(s, kvh, per, d)[place].permute(0, 2, 1, 3, 4).reshape(groups, kvh, -1, d)
    first = (rows @ keys) * st["scale"]
    first = first.masked_fill(t >= prefix[:, None, None, None], float("-inf"))  # [G, KVH, N * per, Lp]
    # What each sequence has behind its prompt.
    group = (torch.arange(s, device=device)[:, None] >= starts[None, 1:]).sum(1)
    u = prefix[group][:, None] + torch.arange(st["tail"], device=device)  # [S, Ls]
    inside = u < context[:, None]
    u = torch.where(inside, u, torch.zeros_like(u))
    slot = tables.gather(1, u // bs) * bs + u % bs
    tail_k = st["k"].view(pages * bs, kvh, d)[slot].float().permute(0, 2, 3, 1).contiguous()
    tail_v = st["v"].view(pages * bs, kvh, d)[slot].float().permute(0, 2, 1, 3).contiguous()
    second = (q.view(s, kvh, per, d) @ tail_k) * st["scale"]
    second = second.masked_fill(~inside[:, None, None, :], float("-inf"))  # [S, KVH, per, Ls]
    # One softmax over both parts.
    index = torch.arange(s, device=device) - starts[group]

    def by_sequence(x):  # [G, KVH, N * per, .] -> [S, KVH, per, .]
        return x.view(groups, kvh, -1, per, x.shape[-1]).permute(0, 2, 1, 3, 4)[group, index]

    top = torch.maximum(by_sequence(first.amax(-1, keepdim=True)), second.amax(-1, keepdim=True))
    grouped = torch.zeros(groups, place.shape[1], kvh, per, 1, device=device)
    grouped[group, index] = top
    e1 = torch.exp(first - grouped.permute(0, 2, 1, 3, 4).reshape(groups, kvh, -1, 1))
    e2 = torch.exp(second - top)
    total = by_sequence(e1.sum(-1, keepdim=True)) + e2.sum(-1, keepdim=True)
    out = (by_sequence(e1 @ values) + e2 @ tail_v) / total
    return out.reshape(s, heads, d).to(st["q"].dtype)


def _own_logprobs(st: dict):
    import cuda_force_amd as cf

    got = cf.token_logprobs(st["logits"], st["tokens"], scale=st["scale"], entropy=st["entropy"], top=st["top"])
    return [v for v in got if v is not None]


def _statistics(st: dict):
    x = st["logits"].detach().float() * st["scale"]
    x = x - x.amax(-1, keepdim=True)
    log_sum = torch.exp(x).sum(-1, keepdim=True).log()
    return x - log_sum


def _plain_logprobs(st: dict):
    logp = _statistics(st)
    tokens = st["tokens"] if st["tokens"].ndim == 2 else st["tokens"][:, None]
    out = [logp.gather(1, tokens).view(st["tokens"].shape)]
    if st["entropy"]:
        out.append(-torch.where(logp == float("-inf"), torch.zeros_like(logp), torch.exp(logp) * logp).sum(-1))
    if st["top"]:
        order = torch.sort(st["logits"], dim=-1, descending=True, stable=True).indices[:, :st["top"]]
        out += [logp.gather(1, order), order]
    return out


def _own_likelihood(st: dict):
    import cuda_force_amd as cf

    got = cf.token_logprobs(st["logits"], st["tokens"], scale=st["scale"], entropy=st["entropy"])
    outputs, grads = [got.logprobs], [st["grad_logprobs"]]
    if st["entropy"]:
        outputs.append(got.entropy)
        grads.append(st["grad_entropy"])
    grad, = torch.autograd.grad(outputs, [st["logits"]], grads)
    return [o.detach() for o in outputs] + [grad]


def _plain_likelihood(st: dict):
    logp = _statistics(st)
    p = torch.exp(logp)
    tokens = st["tokens"] if st["tokens"].ndim == 2 else st["tokens"][:, None]
    given = tokens >= 0
    at = tokens.clamp(min=0)
    out = [torch.where(given, logp.gather(1, at), torch.zeros_like(p[:, :1])).view(st["tokens"].shape)]
    g = torch.where(given, st["grad_logprobs"].view(tokens.shape), torch.zeros_like(p[:, :1]))
    grad = -g.sum(-1, keepdim=True) * p
    if st["entropy"]:
        entropy = -(p * logp).sum(-1)
        out.append(entropy)
        grad -= st["grad_entropy"][:, None] * p * (logp + entropy[:, None])
    grad.scatter_add_(1, at, g)
    return out + [(st["scale"] * grad).to(st["logits"].dtype)]


def _own_fork(st: dict):
    import cuda_force_amd as cf

    status = cf.cache_fork(st["caches"], st["counts"], st["tables"], st["context"], st["parents"], st["children"])
    slots = cf.cache_extend(st["counts"], st["tables"], st["context"], st["children"], st["block"])
    lengths = st["context"].clone()
    cf.cache_release(st["counts"], st["tables"], st["context"], st["children"], st["block"])
    return [status, slots, lengths, st["tables"], st["counts"], st["context"], *st["caches"]]


def _plain_fork(st: dict):
    """Every pair is good and the pool holds enough: what is left is the order
    in which free pages are handed out."""
    counts, tables, context, bs = st["counts"], st["tables"], st["context"], st["block"]
    parents, children = st["parents"].long(), st["children"].long()
    width = tables.shape[1]
    # Fork: whole pages shared, a partial last page copied.
    length = context[parents].long()
    partial = length % bs > 0
    fresh = (counts <= 0).nonzero().view(-1)
    page = fresh[(torch.cumsum(partial, 0) - 1).clamp(min=0)]
    rows = tables[parents].long()
    last = rows.gather(1, ((length - 1) // bs)[:, None])[:, 0]
    inside = torch.arange(width, device=rows.device) < ((length + bs - 1) // bs)[:, None]
    whole = torch.arange(width, device=rows.device) < (length // bs)[:, None]
    counts.index_add_(0, rows[whole], torch.ones_like(rows[whole], dtype=torch.int32))
    rows.scatter_(1, ((length - 1) // bs)[:, None], torch.where(partial, page, last)[:, None])
    tables[children] = torch.where(inside, rows, tables[children].long()).to(torch.int32)
    counts[page[partial]] = 1
    context[children] = length.to(torch.int32)
    valid = torch.arange(bs, device=rows.device) < (length % bs)[:, None]  # [n, block]
    source = (last[:, None] * bs + torch.arange(bs, device=rows.device))[valid]
    target = (page[:, None] * bs + torch.arange(bs, device=rows.device))[valid]
    for cache in st["caches"]:
        flat = cache.view(-1, *cache.shape[2:])
        flat[target] = flat[source]
    status = torch.zeros_like(st["children"])
    # Extend by one token.
    needs = length % bs == 0
    fresh = (counts <= 0).nonzero().view(-1)
    page = fresh[(torch.cumsum(needs, 0) - 1).clamp(min=0)]
    tables[children[needs], length[needs] // bs] = page[needs].to(torch.int32)
    counts[page[needs]] = 1
    context[children] += 1
    slots = tables[children].long().gather(1, (length // bs)[:, None]) * bs + (length % bs)[:, None]
    lengths = context.clone()
    # Release.
    inside = torch.arange(width, device=rows.device) < ((context[children].long() + bs - 1) // bs)[:, None]
    freed = tables[children].long()[inside]
    counts.index_add_(0, freed, torch.full_like(freed, -1, dtype=torch.int32))
    context[children] = 0
    return [status, slots, lengths, tables, counts, context, *st["caches"]]


def _own_copy(st: dict):
    import cuda_force_amd as cf

    return [cf.cache_copy(st["caches"], st["src"], st["dst"]), *st["caches"]]


def _plain_copy(st: dict):
    src, dst = st["src"].long(), st["dst"].long()
    for cache in st["caches"]:
        cache[dst] = cache[src]
    return [torch.zeros_like(st["src"]), *st["caches"]]


def _own_compact(st: dict):
    import cuda_force_amd as cf

    return [*cf.cache_compact(st["caches"], st["counts"], st["tables"], st["context"]), *st["caches"]]


def _plain_compact(st: dict):
    counts, tables, context = st["counts"], st["tables"], st["context"].long()
    bs = st["caches"][0].shape[1]
    live = counts > 0
    number = live.sum()
    index = torch.arange(counts.numel(), device=counts.device)
    holes = (~live & (index < number)).nonzero().view(-1)
    movers = (live & (index >= number)).nonzero().view(-1)
    new_place = index.clone()
    new_place[movers] = holes
    for cache in st["caches"]:
        cache[holes] = cache[movers]
    new_counts = torch.where(live & (index < number), counts, torch.zeros_like(counts))
    new_counts[holes] = counts[movers]
    inside = torch.arange(tables.shape[1], device=tables.device) < ((context + bs - 1) // bs)[:, None]
    new_tables = torch.where(inside, new_place[tables.long()].to(torch.int32), tables)
    return [new_counts, new_tables, number.to(torch.int32).view(1), *st["caches"]]


_OWN = {"attention": _own_attention, "logprobs": _own_logprobs, "likelihood": _own_likelihood, "fork": _own_fork,
        "copy": _own_copy, "compact": _own_compact}
_PLAIN = {"attention": _plain_attention, "logprobs": _plain_logprobs, "likelihood": _plain_likelihood,
          "fork": _plain_fork, "copy": _plain_copy, "compact": _plain_compact}


# ---------------------------------------------------------------------------
# What a pass cannot do without.
# ---------------------------------------------------------------------------


def work(case: dict) -> dict:
    kind, size = case["kind"], _SIZE[case["dtype"]]
    if kind == "attention":
        starts, prefix, member, context = _groups(case)
        once = sum(prefix) + sum(c - prefix[m] for c, m in zip(context, member))
        entries = sum((c + case["block"] - 1) // case["block"] for c in context)
        rows = case["sequences"] * case["heads"] * case["dim"]
        return {"bytes": once * case["kv_heads"] * case["dim"] * 2 * size + 2 * rows * size + 4 * entries,
                "flops": 4 * sum(context) * case["heads"] * case["dim"]}
    if kind in ("logprobs", "likelihood"):
        cells = case["rows"] * case["vocab"]
        small = case["rows"] * (12 * case["count"] + 4 * case["entropy"] + 12 * case.get("top", 0))
        passes = 1 if kind == "logprobs" else 2
        return {"bytes": passes * cells * size + small, "flops": 6 * passes * cells}
    token = case["heads"] * case["dim"] * size * 2 * case["layers"]
    if kind == "fork":
        width, pages = _fork_pages(case)
        lengths = [c for c in _lengths(case["parents"], case["context"]) for _ in range(case["each"])]
        entries = sum((c + case["block"] - 1) // case["block"] for c in lengths)
        return {"bytes": 2 * token * sum(c % case["block"] for c in lengths) + 16 * entries + 4 * pages,
                "flops": entries}
    if kind == "copy":
        return {"bytes": 2 * token * case["block"] * case["pairs"] + 8 * case["pairs"], "flops": case["pairs"]}
    pages = 2 * sum((c + case["block"] - 1) // case["block"] for c in _lengths(case["sequences"], case["context"]))
    # About half of the pool is live, and half of that lies behind the front.
    return {"bytes": 2 * token * case["block"] * (pages // 4) + 8 * pages + 4 * pages, "flops": pages}


# ---------------------------------------------------------------------------
# The definitions in 64 bits.
# ---------------------------------------------------------------------------


def exact(case: dict, seed: int):
    return _EXACT[case["kind"]](prepare(case, seed))


def _exact_attention(st: dict):
    """Sequence by sequence over its whole context, no prompt shared."""
    s, heads, d = st["q"].shape
    kvh, bs = st["k"].shape[2], st["k"].shape[1]
    out = []
    for i, c in enumerate(st["context"].tolist()):
        pages = st["tables"][i, :(c + bs - 1) // bs].long()
        k, v = (st[x][pages].reshape(-1, kvh, d)[:c].double().transpose(0, 1).contiguous() for x in "kv")
        q = st["q"][i].double().view(kvh, heads // kvh, d)
        weights = torch.softmax(torch.bmm(q, k.transpose(1, 2).contiguous()) * st["scale"], -1)
        out.append(torch.bmm(weights, v).view(heads, d))
    return torch.stack(out)


def _exact_logprobs(st: dict):
    logits = st["logits"].detach()
    parts: list[list[torch.Tensor]] = []
    for begin in range(0, logits.shape[0], 128):
        rows = logits[begin:begin + 128].double() * st["scale"]
        logp = rows - torch.logsumexp(rows, -1, keepdim=True)
        tokens = st["tokens"][begin:begin + 128]
        at = tokens.view(rows.shape[0], -1).clamp(min=0)
        picked = torch.gather(logp, 1, at).masked_fill(tokens.view(at.shape) < 0, 0.0)
        got = [picked.view(tokens.shape)]
        if st["entropy"]:
            got.append(torch.special.entr(torch.exp(logp)).sum(-1))
        if st["kind"] == "likelihood":
            g = st["grad_logprobs"][begin:begin + 128].double().view(at.shape)
            leaf = rows.clone().requires_grad_(True)
            lp = torch.log_softmax(leaf, -1)
            loss = (lp.gather(1, at) * g * (tokens.view(at.shape) >= 0)).sum()
            if st["entropy"]:
                loss = loss - ((lp.exp() * lp).sum(-1) * st["grad_entropy"][begin:begin + 128].double()).sum()
            got.append(torch.autograd.grad(loss, leaf)[0] * st["scale"])
        elif st["top"]:
            # A row's order by value, then by index: two sorts, the later one stable.
            best = torch.argsort(-logits[begin:begin + 128].double(), dim=-1, stable=True)[:, :st["top"]]
            got += [torch.gather(logp, 1, best), best]
        parts.append(got)
    return [torch.cat(x) for x in zip(*parts)]


def _exact_fork(st: dict):
    """One pair after the other, on lists."""
    counts, tables, context = (st[x].tolist() for x in ("counts", "tables", "context"))
    bs, caches = st["block"], [c.double() for c in st["caches"]]
    children = st["children"].tolist()

    def fresh():
        page = next(p for p, c in enumerate(counts) if c <= 0)
        counts[page] = 1
        return page

    for parent, child in zip(st["parents"].tolist(), children):
        n = context[parent]
        for i in range(n // bs):
            tables[child][i] = tables[parent][i]
            counts[tables[parent][i]] += 1
        if n % bs:
            old, page = tables[parent][n // bs], fresh()
            tables[child][n // bs] = page
            for cache in caches:
                cache[page, :n % bs] = cache[old, :n % bs]
        context[child] = n
    slots = []
    for child in children:
        if context[child] % bs == 0:
            tables[child][context[child] // bs] = fresh()
        slots.append([tables[child][context[child] // bs] * bs + context[child] % bs])
        context[child] += 1
    lengths = list(context)
    for child in children:
        for i in range((context[child] + bs - 1) // bs):
            counts[tables[child][i]] -= 1
        context[child] = 0
    whole = [torch.tensor(v, dtype=torch.int64) for v in ([0] * len(children), slots, lengths, tables, counts, context)]
    return [*whole, *caches]


def _exact_copy(st: dict):
    caches = [c.double() for c in st["caches"]]
    for cache in caches:
        cache[st["dst"].long()] = cache[st["src"].long()].clone()
    return [torch.zeros_like(st["src"]), *caches]


def _exact_compact(st: dict):
    counts, tables, context = (st[x].tolist() for x in ("counts", "tables", "context"))
    caches = [c.double() for c in st["caches"]]
    bs = caches[0].shape[1]
    live = sum(c > 0 for c in counts)
    holes = [p for p in range(live) if counts[p] <= 0]
    movers = [p for p in range(live, len(counts)) if counts[p] > 0]
    moved = dict(zip(movers, holes))
    for cache in caches:
        cache[holes] = cache[movers].clone()
    for old, new in moved.items():
        counts[new], counts[old] = counts[old], 0
    for row, n in zip(tables, context):
        for i in range((n + bs - 1) // bs):
            row[i] = moved.get(row[i], row[i])
    return [torch.tensor(counts), torch.tensor(tables), torch.tensor([live]), *caches]


_EXACT = {"attention": _exact_attention, "logprobs": _exact_logprobs, "likelihood": _exact_logprobs,
          "fork": _exact_fork, "copy": _exact_copy, "compact": _exact_compact}
