"""The operators of serving in eight bits, as measurable cases.

Each case is a plain dict: ``kind`` names the operator, the rest its sizes.
``run`` with ``own`` false computes it from elementary torch operations, with
``own`` true through the package's entry points.

Kinds:

* ``cache``     keys and values of new tokens written into a paged cache of 8-bit
                codes (a scale for each token and head) and read back;
* ``attention`` causal attention of chunks of new tokens, of single tokens, or of
                both in one batch, over a paged cache of the query's type or of
                8-bit codes;
* ``linear``    activations quantised to 8-bit integers with a scale for each
                token, times 8-bit weights with a scale for each channel.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
#: Codes of a cache: their type and the largest one.
_CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def listed() -> list[dict]:
    return [
        # A decoding step's new tokens, one of each sequence: the latency case.
        {"name": "cache_step", "kind": "cache", "dtype": "bf16", "cache": "int8", "tokens": 64, "kv_heads": 8,
         "dim": 128, "block": 16},
        # A prompt's chunk stored in full.
        {"name": "cache_prompt", "kind": "cache", "dtype": "bf16", "cache": "e4m3", "tokens": 8192, "kv_heads": 8,
         "dim": 128, "block": 16},
        # A chat server's decoding step over a cache of codes.
        {"name": "attention_step", "kind": "attention", "dtype": "bf16", "cache": "int8", "sequences": 64,
         "chunked": 0, "chunk": 1, "idle": 0, "pad": 0, "context": 4096, "heads": 32, "kv_heads": 8, "dim": 128,
         "block": 16},
        # A prompt in one piece, nothing before it.
        {"name": "attention_prompt", "kind": "attention", "dtype": "bf16", "cache": "same", "sequences": 1,
         "chunked": 1, "chunk": 2048, "idle": 0, "pad": 0, "context": 2048, "heads": 32, "kv_heads": 8, "dim": 128,
         "block": 16},
        # The last chunk of a long document: the largest.
        {"name": "attention_document", "kind": "attention", "dtype": "bf16", "cache": "same", "sequences": 1,
         "chunked": 1, "chunk": 2048, "idle": 0, "pad": 0, "context": 32768, "heads": 32, "kv_heads": 8, "dim": 128,
         "block": 32},
        # A server's step: some prompts' chunks next to sequences that decode, in a batch of fixed size.
        {"name": "attention_mixed", "kind": "attention", "dtype": "bf16", "cache": "e4m3", "sequences": 48,
         "chunked": 3, "chunk": 512, "idle": 4, "pad": 77, "context": 4000, "heads": 32, "kv_heads": 8, "dim": 128,
         "block": 16},
        # Short answers scored behind their questions, every query head with its own keys.
        {"name": "attention_ragged", "kind": "attention", "dtype": "f16", "cache": "int8", "sequences": 7,
         "chunked": 7, "chunk": 333, "idle": 0, "pad": 0, "context": 1501, "heads": 16, "kv_heads": 16, "dim": 64,
         "block": 16},
        # The same in full precision.
        {"name": "attention_f32", "kind": "attention", "dtype": "f32", "cache": "same", "sequences": 4, "chunked": 4,
         "chunk": 100, "idle": 0, "pad": 0, "context": 1000, "heads": 32, "kv_heads": 8, "dim": 128, "block": 16},
        # Eight sequences decoding, a block's MLP projection.
        {"name": "linear_step", "kind": "linear", "dtype": "bf16", "rows": 8, "inputs": 4096, "outputs": 11008,
         "bias": False},
        # A mid-sized batch of odd size, a square projection with a bias.
        {"name": "linear_batch", "kind": "linear", "dtype": "f16", "rows": 333, "inputs": 4096, "outputs": 4096,
         "bias": True},
        # The fused adapter linear's benchmark shape.
        {"name": "linear_square", "kind": "linear", "dtype": "bf16", "rows": 8192, "inputs": 4096, "outputs": 4096,
         "bias": False},
        # The MLP's way back at a training batch's number of tokens.
        {"name": "linear_down", "kind": "linear", "dtype": "bf16", "rows": 4096, "inputs": 11008, "outputs": 4096,
         "bias": False},
    ]


def _log(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    kind = rng.choice(["cache"] * 3 + ["attention"] * 6 + ["linear"] * 3)
    if kind == "cache":
        return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "cache": rng.choice(["int8", "e4m3", "same"]), "tokens": _log(rng, 1, 8192),
                "kv_heads": rng.choice([1, 4, 8, 16]), "dim": rng.choice([64, 80, 128, 128, 256]),
                "block": rng.choice([16, 16, 32, 64])}
    if kind == "attention":
        heads, kv_heads = rng.choice([(32, 8), (32, 32), (16, 16), (32, 4), (24, 8), (64, 8), (12, 12)])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
        sequences = _log(rng, 1, 64)
        chunked = rng.choice([0, 1, rng.randint(0, sequences), sequences])
        chunk = _log(rng, 2, 2048) if chunked else 1
        # Padded to the longest, the scores of all sequences stay within 2^30 values.
        most = 2**30 // (sequences * chunk * heads)
        chunk = chunk if most >= 64 else max(1, 2**30 // (sequences * 64 * heads))
        context = _log(rng, 1, max(64, min(16384, most)))
        return {"kind": kind, "dtype": dtype, "cache": rng.choice(["int8", "e4m3", "same"]), "sequences": sequences,
                "chunked": chunked, "chunk": chunk, "idle": rng.choice([0, 0, rng.randint(0, sequences // 4)]),
                "pad": rng.choice([0, 0, rng.randint(1, 50)]), "context": max(context, chunk), "heads": heads,
                "kv_heads": kv_heads, "dim": rng.choice([64, 128, 128, 80, 256]),
                "block": rng.choice([16, 16, 32, 64])}
    sizes = [1024, 2048, 4096, 4096, 11008]
    case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "rows": _log(rng, 1, 8192),
            "inputs": rng.choice([*sizes, 16 * _log(rng, 4, 512)]), "outputs": rng.choice([*sizes, _log(rng, 100, 8192)]),
            "bias": rng.random() < 0.3}
    case["rows"] = max(1, min(case["rows"], 2**37 // (case["inputs"] * case["outputs"])))
    return case


# ---------------------------------------------------------------------------
# Sizes that follow from a case alone.
# ---------------------------------------------------------------------------


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(new tokens, context with them) of each sequence: ragged chunks first,
    then single tokens, then sequences that have none this time."""
    new, context = [], []
    for k in range(case["sequences"]):
        n = case["chunk"] - (k * 131) % (case["chunk"] // 4 + 1) if k < case["chunked"] else 1
        n = 0 if k >= case["sequences"] - case["idle"] else n
        new.append(n)
        context.append(max(n, case["context"] - (k * 7919) % (case["context"] // 2 + 1)))
    return new, context


# ---------------------------------------------------------------------------
# Inputs.
# ---------------------------------------------------------------------------


class _Inputs:
    """Seeded values on the GPU."""

    def __init__(self, seed: int) -> None:
        self.gen = torch.Generator(device="cuda").manual_seed(1_000_003 * (seed % 1_000_003) + 31)

    def normal(self, *shape: int, std: float = 1.0, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return torch.randn(*shape, generator=self.gen, device="cuda").mul_(std).to(dtype)

    def order(self, count: int) -> torch.Tensor:
        return torch.randperm(count, generator=self.gen, device="cuda")


def _i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _quantised(x: torch.Tensor, cache: str, wide: torch.dtype = torch.float64) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes as numbers of the type `wide`, scales): the largest magnitude of
    the last dimension takes the largest code, and every value the nearest one."""
    dtype, top = _CODES[cache]
    scales = x.float().abs().amax(-1) / top
    scales = torch.where(scales > 0, scales, torch.ones_like(scales))
    quotient = x.to(wide) / scales[..., None].to(wide)
    if dtype == torch.int8:
        return quotient.round(), scales
    # Three bits behind the leading one, in steps of 2^-9 at least; ties to even.
    _, exponent = torch.frexp(quotient)
    return torch.ldexp(torch.ldexp(quotient, step := 4 - exponent.clamp(min=-5)).round(), -step), scales


def prepare(case: dict, seed: int) -> dict:
    return _PREPARE[case["kind"]](case, _Inputs(seed))


def _activations(inputs: _Inputs, *shape: int, dtype: torch.dtype) -> torch.Tensor:
    """Normal values of rows of differing size, a few channels far larger."""
    x = inputs.normal(*shape)
    x *= torch.exp(inputs.normal(*shape[:-1], 1, std=0.5))
    x *= 1.0 + 8.0 * (inputs.order(shape[-1]) < max(1, shape[-1] // 64))
    return x.to(dtype)


def _prepare_cache(case: dict, inputs: _Inputs) -> dict:
    dtype, tokens, block = _DTYPES[case["dtype"]], case["tokens"], case["block"]
    pages = 2 * ((tokens + block - 1) // block) + 1
    shape = (pages, block, case["kv_heads"], case["dim"])
    # The keys and values of a fused projection: columns of one tensor, next to
    # the queries' of as many heads.
    fused = _activations(inputs, tokens, 3 * case["kv_heads"], case["dim"], dtype=dtype)
    state = {"kind": "cache", "cache": case["cache"], "dtype": dtype, "keys": fused[:, case["kv_heads"]:2 * case["kv_heads"]],
             "values": fused[:, 2 * case["kv_heads"]:]}
    # Whole pages in any order where a prompt is stored, single places in a step.
    if tokens >= 4 * block:
        t = torch.arange(tokens, device="cuda")
        state["slots"] = inputs.order(pages)[t // block] * block + t % block
    else:
        state["slots"] = inputs.order(pages * block)[:tokens].contiguous()
    if tokens > 8:
        state["slots"][tokens // 2] = -1  # a row that found no page
    code = _CODES[case["cache"]][0] if case["cache"] != "same" else dtype
    for x in "kv":
        state[x + "_cache"] = torch.zeros(shape, device="cuda").to(code)
        state[x + "_scales"] = torch.ones(shape[:3], device="cuda") if case["cache"] != "same" else None
    return state


def _prepare_attention(case: dict, inputs: _Inputs) -> dict:
    dtype = _DTYPES[case["dtype"]]
    bs, kvh, d = case["block"], case["kv_heads"], case["dim"]
    new, context = _lengths(case)
    needs = [(c + bs - 1) // bs for c in context]
    order = inputs.order(sum(needs) + 1).to(torch.int32).cpu()
    tables = torch.zeros(len(new), max(needs), dtype=torch.int32)
    used, starts = 0, [0]
    for k, need in enumerate(needs):
        tables[k, :need] = order[used:used + need]
        used += need
        starts.append(starts[-1] + new[k])
    shape = (used + 1, bs, kvh, d)
    state = {"kind": "attention", "cache": case["cache"], "q": inputs.normal(starts[-1] + case["pad"], case["heads"], d, dtype=dtype),
             "starts": _i32(starts), "tables": tables.cuda(), "context": _i32(context), "scale": 1.0 / math.sqrt(d),
             "most": max(new), "longest": max(context)}
    for x in "kv":
        if case["cache"] == "same":
            state[x], state[x + "_scales"] = inputs.normal(*shape, dtype=dtype), None
        else:
            codes, state[x + "_scales"] = _quantised(inputs.normal(*shape) * torch.exp(inputs.normal(*shape[:3], 1, std=0.5)),
                                                     case["cache"], torch.float32)
            state[x] = codes.to(_CODES[case["cache"]][0])
    return state


def _prepare_linear(case: dict, inputs: _Inputs) -> dict:
    dtype, rows, n, k = _DTYPES[case["dtype"]], case["rows"], case["outputs"], case["inputs"]
    codes, scales = _quantised(inputs.normal(n, k, std=0.02), "int8", torch.float32)
    return {"kind": "linear", "dtype": dtype, "x": _activations(inputs, rows, k, dtype=dtype), "w": codes.to(torch.int8),
            "w_scales": scales, "bias": inputs.normal(n, dtype=dtype) if case["bias"] else None}


_PREPARE = {"cache": _prepare_cache, "attention": _prepare_attention, "linear": _prepare_linear}


# ---------------------------------------------------------------------------
# One pass.
# ---------------------------------------------------------------------------


def run(state: dict):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


def _own_cache(st: dict):
    import cuda_force_amd as cf

    cf.cache_write(st["keys"], st["values"], st["k_cache"], st["v_cache"], st["slots"], st["k_scales"], st["v_scales"])
    return [*cf.cache_read(st["k_cache"], st["v_cache"], st["slots"], st["k_scales"], st["v_scales"], dtype=st["dtype"]),
            *(st[x] for x in ("k_scales", "v_scales") if st[x] is not None)]


def _plain_cache(st: dict):
    slots = st["slots"]
    there = slots >= 0
    at = slots[there]
    back, scales = [], []
    for x, name in (("k", "keys"), ("v", "values")):
        flat = st[x + "_cache"].view(-1, *st[x + "_cache"].shape[2:])
        if st["cache"] == "same":
            flat[at] = st[name][there]
            got = flat[slots.clamp(min=0)].float()
        else:
            codes, s = _quantised(st[name][there], st["cache"])
            st[x + "_scales"].view(-1, s.shape[1])[at] = s
            raw = flat.view(torch.int8)  # indexing knows no type of 8 bits but integers
            raw[at] = codes.to(flat.dtype).view(torch.int8)
            got = raw[slots.clamp(min=0)].view(flat.dtype).float()
            got = got * st[x + "_scales"].view(-1, s.shape[1])[slots.clamp(min=0)][..., None]
            scales.append(st[x + "_scales"])
        back.append(got.masked_fill(~there[:, None, None], 0.0).to(st["dtype"]))
    return back + scales


def _own_attention(st: dict):
    import cuda_force_amd as cf

    return cf.paged_attention_chunk(st["q"], st["k"], st["v"], st["starts"], st["tables"], st["context"],
                                    st["k_scales"], st["v_scales"], scale=st["scale"])


def _plain_attention(st: dict):
    q, starts, context, tables = st["q"].float(), st["starts"].long(), st["context"].long(), st["tables"].long()
    tokens, heads, d = q.shape
    pages, bs, kvh, _ = st["k"].shape
    sequences = context.numel()
    device = q.device
    # The sequences' rows, padded to the most: [S, N].
    new = starts[1:] - starts[:-1]
    i = torch.arange(st["most"], device=device)
    place = torch.where(i < new[:, None], starts[:-1, None] + i, torch.full_like(starts[:-1, None] + i, tokens))
    rows = torch.cat([q, torch.zeros_like(q[:1])])[place]  # [S, N, H, D]
    rows = rows.view(sequences, -1, kvh, heads // kvh, d).permute(0, 2, 1, 3, 4).reshape(sequences, kvh, -1, d)
    t = torch.arange(st["longest"], device=device)
    slot = tables[:, t // bs] * bs + t % bs  # [S, L]

    def gathered(x):  # [S, L, KVH, D]
        flat = st[x].view(pages * bs, kvh, d)
        if st["cache"] == "same":
            return flat[slot].float()
        codes = flat.view(torch.int8)[slot].view(flat.dtype).float()
        return codes * st[x + "_scales"].view(pages * bs, kvh)[slot][..., None]

    scores = (rows @ gathered("k").permute(0, 2, 3, 1).contiguous()).mul_(st["scale"])  # [S, KVH, N * per, L]
    last = (context - new)[:, None] + i  # the position of each row
    hidden = (t > last[..., None]).repeat_interleave(heads // kvh, 1)  # [S, N * per, L]
    scores.masked_fill_(hidden[:, None], float("-inf"))
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    out = (scores @ gathered("v").permute(0, 2, 1, 3).contiguous()) / scores.sum(-1, keepdim=True)
    out = out.view(sequences, kvh, -1, heads // kvh, d).permute(0, 2, 1, 3, 4).reshape(-1, heads, d)
    whole = torch.zeros(tokens + 1, heads, d, device=device)
    whole[place.view(-1)] = out
    return whole[:tokens].to(st["q"].dtype)


def _own_linear(st: dict):
    import cuda_force_amd as cf

    codes, scales = cf.quantize_int8_rows(st["x"])
    return cf.matmul_int8(codes, st["w"], scales, st["w_scales"], bias=st["bias"], dtype=st["dtype"])


def _plain_linear(st: dict):
    codes, scales = _quantised(st["x"], "int8")
    y = (codes.float() @ st["w"].float().t()) * scales[:, None] * st["w_scales"]
    if st["bias"] is not None:
        y = y + st["bias"].float()
    return y.to(st["dtype"])


_OWN = {"cache": _own_cache, "attention": _own_attention, "linear": _own_linear}
_PLAIN = {"cache": _plain_cache, "attention": _plain_attention, "linear": _plain_linear}


# ---------------------------------------------------------------------------
# What a pass cannot do without.
# ---------------------------------------------------------------------------


def work(case: dict) -> dict:
    size = _SIZE[case["dtype"]]
    held = size if case.get("cache") == "same" else 1  # bytes of a value in the cache
    if case["kind"] == "cache":
        cells = 2 * case["tokens"] * case["kv_heads"]
        row = case["dim"] * held + (4 if held == 1 else 0)
        # Given values read, codes written, codes read, values written.
        return {"bytes": 2 * cells * (case["dim"] * size + row) + 16 * case["tokens"], "flops": 4 * cells * case["dim"]}
    if case["kind"] == "attention":
        new, context = _lengths(case)
        read = sum(c for n, c in zip(new, context) if n) * case["kv_heads"] * 2
        rows = (sum(new) + case["pad"]) * case["heads"] * case["dim"]
        seen = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(new, context))
        return {"bytes": read * (case["dim"] * held + (4 if case["cache"] != "same" else 0)) + 2 * rows * size,
                "flops": 4 * seen * case["heads"] * case["dim"]}
    m, n, k = case["rows"], case["outputs"], case["inputs"]
    return {"bytes": m * k * size + n * k + m * n * size + 4 * n + (n * size if case["bias"] else 0),
            "flops": 2 * m * n * k}


# ---------------------------------------------------------------------------
# The definitions in 64 bits.
# ---------------------------------------------------------------------------


def exact(case: dict, seed: int):
    return _EXACT[case["kind"]](prepare(case, seed))


def _steps(x: torch.Tensor, cache: str) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes in float64, scales): by the list of all magnitudes that a code has."""
    dtype, top = _CODES[cache]
    if dtype == torch.int8:
        grid = torch.arange(128, dtype=torch.float64, device=x.device)
    else:
        grid = torch.tensor([(8 * (e > 0) + m) * 2.0 ** (max(e, 1) - 10) for e in range(16) for m in range(8)][:127],
                            dtype=torch.float64, device=x.device)
    scales = (x.double().abs().amax(-1).float() / top)
    scales[scales == 0] = 1.0
    size = (x.double() / scales.double().unsqueeze(-1)).abs()
    above = torch.searchsorted(grid, size).clamp(1, grid.numel() - 1)
    low, high = grid[above - 1], grid[above]
    down, up = size - low, high - size
    even = (above - 1) % 2 == 0
    return torch.where((down < up) | ((down == up) & even), low, high) * torch.sign(x.double()), scales


def _exact_cache(st: dict):
    out, scales = [], []
    there = [(i, s) for i, s in enumerate(st["slots"].tolist()) if s >= 0]
    rows = torch.tensor([i for i, _ in there], device="cuda")
    at = torch.tensor([s for _, s in there], device="cuda")
    for x, name in (("k", "keys"), ("v", "values")):
        given = st[name].double()
        back = torch.zeros_like(given)
        if st["cache"] == "same":
            back[rows] = given[rows]
        else:
            codes, s = _steps(st[name], st["cache"])
            back[rows] = (codes * s.double().unsqueeze(-1))[rows]
            whole = st[x + "_scales"].double().flatten(0, 1)
            whole[at] = s[rows].double()
            scales.append(whole.view(st[x + "_scales"].shape))
        out.append(back)
    return out + scales


def _exact_attention(st: dict):
    """Sequence by sequence, a head at a time."""
    heads, d = st["q"].shape[1:]
    kvh, bs = st["k"].shape[2], st["k"].shape[1]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    starts = st["starts"].tolist()
    for s, c in enumerate(st["context"].tolist()):
        first, end = starts[s], starts[s + 1]
        if first == end:
            continue
        pages = st["tables"][s, :(c + bs - 1) // bs].long()
        k, v = (st[x].view(torch.uint8)[pages].view(st[x].dtype).flatten(0, 1)[:c].double() for x in "kv")
        if st["cache"] != "same":
            k, v = (t * st[x][pages].flatten(0, 1)[:c].double().unsqueeze(-1) for t, x in ((k, "k_scales"), (v, "v_scales")))
        seen = torch.ones(end - first, c, dtype=torch.bool, device="cuda").tril(c - (end - first))
        for h in range(heads):
            own_head = h * kvh // heads
            scores = torch.mm(st["q"][first:end, h].double(), k[:, own_head].t().contiguous()) * st["scale"]
            weights = torch.softmax(torch.where(seen, scores, -math.inf), -1)
            out[first:end, h] = torch.mm(weights, v[:, own_head].contiguous())
    return out


def _exact_linear(st: dict):
    codes, scales = _steps(st["x"], "int8")
    y = torch.mm(codes, st["w"].double().t().contiguous()) * torch.outer(scales.double(), st["w_scales"].double())
    return y if st["bias"] is None else torch.add(y, st["bias"].double())


_EXACT = {"cache": _exact_cache, "attention": _exact_attention, "linear": _exact_linear}
