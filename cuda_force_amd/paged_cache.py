"""Operators over a paged KV cache.

The layouts are those of paged attention (cuda/include/cudaforge/paged_attention.cuh:10-61):
a cache is ``[pages, block, kv_heads, head_dim]``; token t of sequence s lies in
page ``block_tables[s, t // block]`` at offset ``t % block``; ``context_lens[s]``
tokens of it are in use. Tables, lengths and counts are int32 tensors on the
caches' device, and every operator works on them there: nothing is read back
and nothing waits.
"""

from __future__ import annotations

import math
from collections.abc import Sequence

import torch

from cuda_force_amd import ops
from cuda_force_amd.ops import KERNEL_DTYPES, _dispatch_available, _refuse_gpu_fallback, _same_dtype


def _check_int32(t: torch.Tensor, dims: int, like: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.ndim != dims:
        raise ValueError(f"{name} must have {dims} dimension(s), got shape {tuple(t.shape)}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")
    return t


def _paged_attention_reference(
    query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
    context_lens: torch.Tensor, scale: float,
) -> torch.Tensor:
    """Sequence by sequence in plain PyTorch (fp32, or fp64 where the cache is)."""
    pages, block, kv_heads, dim = k_cache.shape
    heads = query.shape[1]
    wide = torch.float64 if query.dtype == torch.float64 else torch.float32
    rows = []
    for s, length in enumerate(context_lens.tolist()):
        token = torch.arange(min(max(length, 0), block_tables.shape[1] * block), device=query.device)
        page = block_tables[s].long()[token // max(block, 1)]
        there = (page >= 0) & (page < pages)
        slot = (page * block + token % max(block, 1))[there]
        if slot.numel() == 0:
            rows.append(torch.zeros(heads, dim, dtype=wide, device=query.device))
            continue
        k = k_cache.reshape(-1, kv_heads, dim)[slot].to(wide).permute(1, 2, 0).contiguous()
        v = v_cache.reshape(-1, kv_heads, dim)[slot].to(wide).permute(1, 0, 2).contiguous()
        scores = (query[s].to(wide).view(kv_heads, -1, dim) @ k) * scale
        none = (scores == float("-inf")).all(-1, keepdim=True)
        rows.append((torch.softmax(scores, -1) @ v).masked_fill(none, 0.0).reshape(heads, dim))
    if not rows:
        return torch.empty_like(query)
    return torch.stack(rows).to(query.dtype)


def paged_attention_shared(
    query: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    group_starts: torch.Tensor,
    prefix_lens: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention of one new token per sequence over a paged cache, for a batch in
    which groups of neighbouring sequences begin with the same tokens.

    ``query`` is ``[sequences, heads, head_dim]``, the caches ``[pages, block,
    kv_heads, head_dim]`` of its dtype (heads a multiple of kv_heads),
    ``block_tables`` ``[sequences, width]`` and ``context_lens``
    ``[sequences]``. Sequences ``group_starts[g] .. group_starts[g + 1] - 1``
    hold the same keys and values in their first ``prefix_lens[g]`` tokens (in
    the same pages, or in copies; a prefix need not fill its last page). Those
    are read once for the whole group, from the first of its sequences whose
    context holds all of them; the result is that of every sequence attending to
    its own table. Sequences that no group holds, or whose context is shorter
    than their group's prefix, are served alone. ``scale`` defaults to
    ``1 / sqrt(head_dim)``.

    Returns ``[sequences, heads, head_dim]``; zeros for an empty context. A
    table entry that names no page leaves its tokens out. fp32, fp16 and bf16;
    not differentiable on the kernels (a call that needs a gradient runs the
    PyTorch composition). Not in the reference's API.

    Raises:
        ValueError: for shapes or devices that do not match, or caches that are
            not contiguous (a copy of a cache is never made).
        TypeError: for integer arguments that are not int32.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(query.shape[-1]) if query.ndim and query.shape[-1] else 1.0
    if ops._DIRECT is not None and not ops._compiling():
        direct = ops._DIRECT.try_paged_attention_shared(
            query, k_cache, v_cache, group_starts, prefix_lens, block_tables, context_lens, scale)
        if direct is not None:
            return direct
    if query.ndim != 3:
        raise ValueError(f"query must be [sequences, heads, head_dim], got shape {tuple(query.shape)}")
    if k_cache.ndim != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(
            f"caches must be [pages, block, kv_heads, head_dim] and alike, got {tuple(k_cache.shape)} "
            f"and {tuple(v_cache.shape)}"
        )
    sequences, heads, dim = query.shape
    if k_cache.shape[3] != dim or k_cache.shape[2] == 0 or heads % k_cache.shape[2]:
        raise ValueError(
            f"query of {heads} heads of {dim} does not fit a cache of {k_cache.shape[2]} heads of {k_cache.shape[3]}"
        )
    if dim > 1024:
        raise ValueError(f"head_dim {dim} is above 1024")
    for cache, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if cache.device != query.device:
            raise ValueError(f"{name} is on {cache.device}, expected {query.device}")
        if not cache.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    starts = _check_int32(group_starts, 1, query, "group_starts").contiguous()
    prefix = _check_int32(prefix_lens, 1, query, "prefix_lens").contiguous()
    tables = _check_int32(block_tables, 2, query, "block_tables").contiguous()
    context = _check_int32(context_lens, 1, query, "context_lens").contiguous()
    if tables.shape[0] != sequences or context.shape[0] != sequences:
        raise ValueError(f"block_tables and context_lens must have {sequences} rows")
    if starts.shape[0] != prefix.shape[0] + 1:
        raise ValueError(
            f"group_starts must have one entry more than prefix_lens, got {starts.shape[0]} and {prefix.shape[0]}"
        )
    query = query.contiguous()
    if (
        _dispatch_available("paged_attention_shared", query, k_cache, v_cache)
        and query.dtype in KERNEL_DTYPES
        and _same_dtype(query, k_cache, v_cache)
    ):
        return torch.ops.cudaforge.paged_attention_shared(
            query, k_cache, v_cache, starts, prefix, tables, context, float(scale))
    if not _same_dtype(query, k_cache, v_cache):
        raise ValueError(f"query and caches differ in dtype: {query.dtype}, {k_cache.dtype}, {v_cache.dtype}")
    _refuse_gpu_fallback("paged_attention_shared", query, k_cache, v_cache)
    return _paged_attention_reference(query, k_cache, v_cache, tables, context, float(scale))


# ---------------------------------------------------------------------------
# Pages. Plain forms first: one entry of a list after the other, in place.
# ---------------------------------------------------------------------------


def _copy_reference(caches: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor) -> torch.Tensor:
    pages = caches[0].shape[0]
    pairs = list(zip(src.tolist(), dst.tolist()))
    owner: dict[int, int] = {}
    named = {d for _, d in pairs}
    for i, (s, d) in enumerate(pairs):
        if 0 <= s < pages and 0 <= d < pages:
            owner.setdefault(d, i)
    status = [0 if owner.get(d) == i and s not in named else 1 for i, (s, d) in enumerate(pairs)]
    good = [i for i, bad in enumerate(status) if not bad]
    if good:
        for cache in caches:
            cache[dst[good].long()] = cache[src[good].long()]
    return torch.tensor(status, dtype=torch.int32, device=src.device)


def _fork_reference(
    caches: Sequence[torch.Tensor], ref_counts: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
    parents: torch.Tensor, children: torch.Tensor,
) -> torch.Tensor:
    pages, block = caches[0].shape[:2]
    sequences, width = block_tables.shape
    lengths = context_lens.tolist()
    counts = ref_counts.tolist()
    free = [p for p, c in enumerate(counts) if c <= 0]
    taken: set[int] = set()
    status = []
    shared: list[int] = []
    out_of_pages = False
    for parent, child in zip(parents.tolist(), children.tolist()):
        ok = 0 <= parent < sequences and 0 <= child < sequences and child not in taken and block > 0
        ok = ok and 0 < lengths[parent] <= width * block and lengths[child] <= 0
        if not ok:
            status.append(1)
            continue
        taken.add(child)
        whole, rest = divmod(lengths[parent], block)
        if rest and (out_of_pages or not free):
            out_of_pages = True
            status.append(2)
            continue
        row = block_tables[parent, :whole]
        block_tables[child, :whole] = row
        shared += [page for page in row.tolist() if 0 <= page < pages]
        if rest:
            page, old = free.pop(0), int(block_tables[parent, whole])
            block_tables[child, whole] = page
            ref_counts[page] = 1
            if 0 <= old < pages:
                for cache in caches:
                    cache[page, :rest] = cache[old, :rest]
        context_lens[child] = lengths[parent]
        status.append(0)
    for page in shared:
        ref_counts[page] += 1
    return torch.tensor(status, dtype=torch.int32, device=parents.device)


def _extend_reference(
    ref_counts: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, sequences: torch.Tensor,
    block_size: int, tokens: int,
) -> torch.Tensor:
    rows, width = block_tables.shape
    pages = ref_counts.shape[0]
    capacity = min(width * block_size, 2**31 - 1)
    free = [p for p, c in enumerate(ref_counts.tolist()) if c <= 0]
    slots = torch.full((sequences.shape[0], tokens), -1, dtype=torch.int64, device=sequences.device)
    seen: set[int] = set()
    wanted = 0  # pages that the entries so far asked for
    given = 0
    total = len(free)
    for i, s in enumerate(sequences.tolist()):
        if not 0 <= s < rows or s in seen:
            continue
        seen.add(s)
        length = max(int(context_lens[s]), 0)
        if length + tokens > capacity:
            continue
        first = -(-length // block_size)
        need = -(-(length + tokens) // block_size) - first
        wanted += need
        if need and wanted > total:
            continue
        for k in range(need):
            page = free[given + k]
            block_tables[s, first + k] = page
            ref_counts[page] = 1
        given += need
        context_lens[s] = length + tokens
        at = torch.arange(length, length + tokens, device=sequences.device)
        page = block_tables[s].long()[at // block_size]
        slots[i] = torch.where((page >= 0) & (page < pages), page * block_size + at % block_size, -1)
    return slots


def _release_reference(
    ref_counts: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, sequences: torch.Tensor,
    block_size: int,
) -> None:
    rows, width = block_tables.shape
    for s in sequences.tolist():
        if not 0 <= s < rows:
            continue
        held = min(-(-max(int(context_lens[s]), 0) // block_size), width)
        context_lens[s] = 0
        for page in block_tables[s, :held].tolist():
            if 0 <= page < ref_counts.shape[0] and ref_counts[page] > 0:
                ref_counts[page] -= 1


def _compact_reference(
    caches: Sequence[torch.Tensor], ref_counts: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    counts = ref_counts.tolist()
    block = caches[0].shape[1]
    live = sum(c > 0 for c in counts)
    holes = [p for p in range(live) if counts[p] <= 0]
    movers = [p for p in range(live, len(counts)) if counts[p] > 0]
    if holes:
        for cache in caches:
            cache[holes] = cache[movers]
    place = dict(zip(movers, holes))
    new_counts = [max(c, 0) if p < live else 0 for p, c in enumerate(counts)]
    for old, new in place.items():
        new_counts[new] = counts[old]
    new_tables = block_tables.clone()
    for s, length in enumerate(context_lens.tolist()):
        held = min(-(-max(length, 0) // max(block, 1)), block_tables.shape[1])
        row = [place.get(p, p) for p in block_tables[s, :held].tolist()]
        new_tables[s, :held] = torch.tensor(row, dtype=torch.int32, device=new_tables.device)
    device = ref_counts.device
    return (torch.tensor(new_counts, dtype=torch.int32, device=device), new_tables,
            torch.tensor([live], dtype=torch.int32, device=device))


if ops._EXTENSION_LOADED:
    _CPU = torch.library.Library("cudaforge", "IMPL")
    for _name, _form in (("cache_copy", _copy_reference), ("cache_fork", _fork_reference),
                         ("cache_extend", _extend_reference), ("cache_release", _release_reference),
                         ("cache_compact", _compact_reference)):
        _CPU.impl(_name, _form, "CPU")


def _check_caches(caches: Sequence[torch.Tensor], dims: int) -> list[torch.Tensor]:
    if isinstance(caches, torch.Tensor) or len(caches) == 0:
        raise ValueError("caches must be a non-empty list of tensors (K and V of every layer)")
    first = caches[0]
    if first.ndim < dims:
        raise ValueError(f"caches must be [pages, block, ...], got shape {tuple(first.shape)}")
    for cache in caches:
        if cache.shape != first.shape or cache.dtype != first.dtype or cache.device != first.device:
            raise ValueError(
                f"caches differ: {tuple(first.shape)} {first.dtype} on {first.device} and "
                f"{tuple(cache.shape)} {cache.dtype} on {cache.device}"
            )
        if not cache.is_contiguous():
            raise ValueError("caches must be contiguous")
        if cache.requires_grad:
            raise ValueError("caches are written in place and may not require gradients")
    return list(caches)


def _check_state(ref_counts: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor) -> None:
    _check_int32(ref_counts, 1, ref_counts, "ref_counts")
    _check_int32(block_tables, 2, ref_counts, "block_tables")
    _check_int32(context_lens, 1, ref_counts, "context_lens")
    if block_tables.shape[0] != context_lens.shape[0]:
        raise ValueError(
            f"block_tables has {block_tables.shape[0]} rows but context_lens {context_lens.shape[0]}")
    for t, name in ((ref_counts, "ref_counts"), (block_tables, "block_tables"), (context_lens, "context_lens")):
        if not t.is_contiguous():  # written in place: never a copy
            raise ValueError(f"{name} must be contiguous")


def _check_pages(caches: Sequence[torch.Tensor], ref_counts: torch.Tensor) -> None:
    if caches[0].shape[0] != ref_counts.shape[0]:
        raise ValueError(f"ref_counts counts {ref_counts.shape[0]} pages, the caches hold {caches[0].shape[0]}")
    if caches[0].device != ref_counts.device:
        raise ValueError(f"ref_counts is on {ref_counts.device}, expected {caches[0].device}")


def _positive(value: int, name: str) -> int:
    if value <= 0:
        raise ValueError(f"{name} must be positive, got {value}")
    return int(value)


def cache_copy(caches: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor) -> torch.Tensor:
    """Copy page ``src[i]`` to page ``dst[i]`` in every cache, all as they were
    before the call.

    ``caches`` are tensors ``[pages, ...]`` of one shape and any dtype, ``src``
    and ``dst`` int32 ``[n]`` on their device. Returns int32 ``[n]``: 0 for a
    copied page, 1 for an entry left out (a page out of range, a ``dst`` that an
    earlier entry whose pages are in range names, or a ``src`` that some entry
    names as its ``dst``). Not in the reference's API.

    Raises:
        ValueError: for caches that differ, are not contiguous or require
            gradients, or lists that differ in length.
        TypeError: for lists that are not int32.
    """
    if ops._DIRECT is not None and not ops._compiling():
        direct = ops._DIRECT.try_cache_copy(caches, src, dst)
        if direct is not None:
            return direct
    caches = _check_caches(caches, 1)
    src = _check_int32(src, 1, caches[0], "src").contiguous()
    dst = _check_int32(dst, 1, caches[0], "dst").contiguous()
    if src.shape != dst.shape:
        raise ValueError(f"src and dst differ in length: {src.shape[0]} and {dst.shape[0]}")
    if _dispatch_available("cache_copy", *caches):
        return torch.ops.cudaforge.cache_copy(caches, src, dst)
    return _copy_reference(caches, src, dst)


def cache_fork(
    caches: Sequence[torch.Tensor], ref_counts: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
    parents: torch.Tensor, children: torch.Tensor,
) -> torch.Tensor:
    """Make row ``children[i]`` of the tables continue from row ``parents[i]``.

    The child gets the parent's length and shares its whole pages (their counts
    in ``ref_counts`` go up); the used tokens of a partial last page are copied
    to the lowest free page (a count <= 0) in every cache, so parent and child
    may both grow. Children must be empty rows (length <= 0), each named once. A
    parent may have many children, but cannot be a child of the same call.

    ``caches`` are ``[pages, block, ...]``, ``ref_counts`` ``[pages]``,
    ``block_tables`` ``[sequences, width]``, ``context_lens`` ``[sequences]``,
    all written in place; ``parents`` and ``children`` int32 ``[n]``. Returns
    int32 ``[n]``: 0 done, 1 left out (a row out of range, an empty parent, a
    child in use or named before), 2 no page was free for it (nor for a later
    entry that needs one). Not in the reference's API.

    Raises:
        ValueError: for shapes, devices or layouts that do not match.
        TypeError: for integer arguments that are not int32.
    """
    if ops._DIRECT is not None and not ops._compiling():
        direct = ops._DIRECT.try_cache_fork(caches, ref_counts, block_tables, context_lens, parents, children)
        if direct is not None:
            return direct
    caches = _check_caches(caches, 2)
    _check_state(ref_counts, block_tables, context_lens)
    _check_pages(caches, ref_counts)
    parents = _check_int32(parents, 1, ref_counts, "parents").contiguous()
    children = _check_int32(children, 1, ref_counts, "children").contiguous()
    if parents.shape != children.shape:
        raise ValueError(f"parents and children differ in length: {parents.shape[0]} and {children.shape[0]}")
    if _dispatch_available("cache_fork", *caches):
        return torch.ops.cudaforge.cache_fork(caches, ref_counts, block_tables, context_lens, parents, children)
    return _fork_reference(caches, ref_counts, block_tables, context_lens, parents, children)


def cache_extend(
    ref_counts: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, sequences: torch.Tensor,
    block_size: int, tokens: int = 1,
) -> torch.Tensor:
    """Make rows ``sequences[i]`` of the tables ``tokens`` longer.

    Rows that need further pages get the lowest free ones, in the order of the
    list; an empty row starts anew. Returns int64 ``[n, tokens]`` slots, ``page *
    block_size + offset``: where the keys and values of the new tokens go in
    ``cache.view(-1, kv_heads, head_dim)``. They are -1 for an entry left out: a
    row out of range or named before, one whose table would overflow, or one for
    which not all pages were free (nor then for a later entry that needs one).
    An index of -1 is the last token of the cache, in whosever page that lies:
    send such tokens elsewhere before storing through the slots, for instance
    ``slots.clamp(min=0)`` to a page 0 whose count the program set to 1 before
    it stored anything. The last page of a row must be its own (``cache_fork``
    sees to that): the new tokens go there. Not in the reference's API.

    Raises:
        ValueError: for shapes, devices or layouts that do not match, or sizes
            that are not positive.
        TypeError: for integer arguments that are not int32.
    """
    if ops._DIRECT is not None and not ops._compiling():
        direct = ops._DIRECT.try_cache_extend(ref_counts, block_tables, context_lens, sequences, block_size, tokens)
        if direct is not None:
            return direct
    _check_state(ref_counts, block_tables, context_lens)
    sequences = _check_int32(sequences, 1, ref_counts, "sequences").contiguous()
    block_size, tokens = _positive(block_size, "block_size"), _positive(tokens, "tokens")
    arguments = (ref_counts, block_tables, context_lens, sequences, block_size, tokens)
    if _dispatch_available("cache_extend", ref_counts):
        return torch.ops.cudaforge.cache_extend(*arguments)
    return _extend_reference(*arguments)


def cache_release(
    ref_counts: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, sequences: torch.Tensor,
    block_size: int,
) -> None:
    """Empty rows ``sequences[i]`` of the tables: their lengths become 0 and the
    counts of their pages go down by one (not below 0; a page at 0 is free).

    Rows out of range are left out, a row named twice is released once, table
    entries stay as they are. Not in the reference's API.

    Raises:
        ValueError: for shapes, devices or layouts that do not match.
        TypeError: for integer arguments that are not int32.
    """
    if ops._DIRECT is not None and not ops._compiling():
        if ops._DIRECT.try_cache_release(ref_counts, block_tables, context_lens, sequences, block_size):
            return
    _check_state(ref_counts, block_tables, context_lens)
    sequences = _check_int32(sequences, 1, ref_counts, "sequences").contiguous()
    block_size = _positive(block_size, "block_size")
    arguments = (ref_counts, block_tables, context_lens, sequences, block_size)
    if _dispatch_available("cache_release", ref_counts):
        torch.ops.cudaforge.cache_release(*arguments)
    else:
        _release_reference(*arguments)


def cache_compact(
    caches: Sequence[torch.Tensor], ref_counts: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Move the live pages (a count > 0) of every cache to its front.

    Of L live pages, number j at or past L goes to free page number j below L;
    pages below L stay. Returns ``(ref_counts, block_tables, live)`` for the
    cache afterwards, ``live`` int32 ``[1]`` holding L: pages from L on may be
    given up. The arguments' counts and tables are left as they were, and stay
    readable until a moved page's old place is used again. Not in the
    reference's API.

    Raises:
        ValueError: for shapes, devices or layouts that do not match.
        TypeError: for integer arguments that are not int32.
    """
    if ops._DIRECT is not None and not ops._compiling():
        direct = ops._DIRECT.try_cache_compact(caches, ref_counts, block_tables, context_lens)
        if direct is not None:
            return direct
    caches = _check_caches(caches, 2)
    _check_state(ref_counts, block_tables, context_lens)
    _check_pages(caches, ref_counts)
    if _dispatch_available("cache_compact", *caches):
        return torch.ops.cudaforge.cache_compact(caches, ref_counts, block_tables, context_lens)
    return _compact_reference(caches, ref_counts, block_tables, context_lens)
