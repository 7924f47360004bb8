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
