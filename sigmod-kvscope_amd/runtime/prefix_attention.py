"""Attention over the paged cache for a batch whose rows share prefixes, and the running attention weight of
every cached token.

Requests of a service begin with the same instructions; their keys and values are in the cache once, in
pages every request of the group points to.  Attention that walks each request's own table reads those
pages once per request.  Here a group's queries read them together, once per tile of query rows, on the
matrix cores, and the result joins the attention over each row's own pages through the logarithms of
their sums.

With ``scores`` the call also adds to every own token the weight it received, the running statistic
that ``runtime.eviction.evict_tokens`` ranks tokens by.
"""

from __future__ import annotations

import ctypes

import torch

import ekv_hip
from observe.allocation import _workspace, check_tensors

_QUERY_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _cache_shape(kv_cache: torch.Tensor) -> tuple[int, int, int, int]:
    """(pages, block size, KV heads, head dim) of a ``[pages, 2, block, kv_heads, dim]`` cache."""
    if not isinstance(kv_cache, torch.Tensor) or kv_cache.ndim != 5 or kv_cache.shape[1] != 2:
        raise ValueError("kv_cache must be a [pages, 2, block, kv_heads, dim] tensor")
    pages, _, block, heads, dim = kv_cache.shape
    if block < 1 or heads < 1:
        raise ValueError(f"a cache of blocks of {block} tokens and {heads} heads is empty")
    if dim > 1 and kv_cache.stride(4) != 1:
        raise ValueError("kv_cache must have contiguous rows")
    return pages, block, heads, dim


def _arguments(query, kv_cache, table, lens, scale, q_start, max_query, prefix_table, prefix_lens, prefix_rows,
               k_scale, v_scale, scores, decay, out, lse):
    pages, block, kv_heads, dim = _cache_shape(kv_cache)
    if not isinstance(query, torch.Tensor) or query.ndim != 3 or query.shape[2] != dim:
        raise ValueError(f"query must be a [tokens, heads, {dim}] tensor")
    if not isinstance(table, torch.Tensor) or table.ndim != 2:
        raise ValueError("the block table must be a [rows, width] tensor")
    tokens, q_heads, _ = query.shape
    rows, width = table.shape
    if tokens == 0:
        query = query.new_empty(query.shape)  # no rows to be contiguous: an empty tensor's strides may be anything
    groups = prefix_width = 0
    if prefix_table is not None:
        if not isinstance(prefix_table, torch.Tensor) or prefix_table.ndim != 2:
            raise ValueError("prefix_table must be a [groups, width] tensor")
        groups, prefix_width = prefix_table.shape
        if prefix_lens is None:
            raise ValueError("a prefix_table needs prefix_lens")
        if prefix_rows is None and groups != 1:
            raise ValueError(f"{groups} prefixes need prefix_rows")
    elif prefix_lens is not None or prefix_rows is not None:
        raise ValueError("prefix_lens and prefix_rows need a prefix_table")
    device = check_tensors(
        ("query", query, _QUERY_TYPES, (tokens, q_heads, dim)),
        ("kv_cache", kv_cache, kv_cache.dtype, kv_cache.shape),
        ("table", table, torch.int32, (rows, width)), ("lens", lens, torch.int32, (rows,)),
        ("q_start", q_start, torch.int32, (rows + 1,)),
        ("prefix_table", prefix_table, torch.int32, (groups, prefix_width)),
        ("prefix_lens", prefix_lens, torch.int32, (groups,)),
        ("prefix_rows", prefix_rows, torch.int32, (groups + 1,)),
        ("out", out, query.dtype, query.shape), ("lse", lse, torch.float32, (tokens, q_heads)))
    if scores is not None:
        if not isinstance(scores, torch.Tensor) or scores.ndim != 3 or scores.shape[:2] != (rows, kv_heads) \
                or scores.shape[2] < width * block:
            raise ValueError(f"scores must be a [{rows}, {kv_heads}, {width * block} or more] tensor")
        if check_tensors(("scores", scores, torch.float32, scores.shape)) != device:
            raise ValueError(f"scores must be on {device}")
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=device)
    if lse is None:
        lse = torch.empty(tokens, q_heads, dtype=torch.float32, device=device)
    elif not lse.is_contiguous():
        raise ValueError("lse must be contiguous")
    a = ekv_hip.Attention()
    a.query, (a.q_stride_token, a.q_stride_head, _) = query.data_ptr(), query.stride()
    stride = kv_cache.stride()
    a.keys = kv_cache.data_ptr()
    a.values = a.keys + stride[1] * kv_cache.element_size() if a.keys else 0
    a.kv_stride_block, a.kv_stride_pos, a.kv_stride_head, a.blocks = stride[0], stride[2], stride[3], pages
    a.table, a.table_stride, a.lens = table.data_ptr(), table.stride(0), lens.data_ptr()
    if q_start is not None:
        a.q_start = q_start.data_ptr()
    if groups and prefix_width:
        a.prefix_table, a.prefix_stride, a.prefix_lens = (prefix_table.data_ptr(), prefix_table.stride(0),
                                                          prefix_lens.data_ptr())
        if prefix_rows is not None:
            a.prefix_rows = prefix_rows.data_ptr()
        a.prefix_groups, a.prefix_width = groups, prefix_width
    if scores is not None:
        a.scores, a.scores_stride_row, a.scores_stride_head = scores.data_ptr(), scores.stride(0), scores.stride(1)
    a.out, (a.out_stride_token, a.out_stride_head, _) = out.data_ptr(), out.stride()
    a.lse = lse.data_ptr()
    a.q_dtype, a.kv_dtype = ekv_hip.dtype_code(query.dtype), ekv_hip.dtype_code(kv_cache.dtype)
    a.rows, a.width, a.tokens, a.max_query = rows, width, tokens, max_query
    a.q_heads, a.kv_heads, a.head_dim, a.block_size = q_heads, kv_heads, dim, block
    a.scale, a.k_scale, a.v_scale, a.decay = scale, k_scale, v_scale, decay
    return a, out, lse, device


def prefix_attention(
    query: torch.Tensor,
    kv_cache: torch.Tensor,
    table: torch.Tensor,
    lens: torch.Tensor,
    scale: float,
    *,
    q_start: torch.Tensor | None = None,
    max_query: int = 1,
    prefix_table: torch.Tensor | None = None,
    prefix_lens: torch.Tensor | None = None,
    prefix_rows: torch.Tensor | None = None,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
    scores: torch.Tensor | None = None,
    decay: float = 1.0,
    out: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    stream=None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """One layer's attention of a batch: ``(out [tokens, q_heads, dim], lse float32 [tokens, q_heads])``.

    ``query [tokens, q_heads, dim]``; ``kv_cache [pages, 2, block, kv_heads, dim]``; ``table`` int32
    ``[rows, width]`` and ``lens`` int32 ``[rows]``: each row's own pages and tokens, the query tokens
    included (a ``DecodeView``'s buffers serve).  Row r's query tokens are ``q_start[r] .. q_start[r + 1]``
    (None: one a row) and the last of its own tokens; query i of t sees slots up to ``len - t + i``.
    ``max_query`` bounds a row's query tokens; what passes it, or is no row's, gets 0 and -inf, as a query
    that sees nothing does.

    ``prefix_table`` int32 ``[groups, pages]`` and ``prefix_lens`` int32 ``[groups]``: shared prefixes, seen
    whole by every query of rows ``prefix_rows[g] .. prefix_rows[g + 1]`` (ascending; None: one group of
    every row).

    ``scores`` float32 ``[rows, kv_heads, slots]``: slot j of each row's tokens becomes ``decay * scores``
    plus the weight its key received from this call's queries.  Types, head dims and limits as
    ``ekv_prefix_attention`` documents them; ``k_scale`` / ``v_scale`` are an fp8 cache's scales.
    ``workspace``: a uint8 device tensor that the call may overwrite (one is allocated if none is given;
    under graph capture it then belongs to the graph's pool).  No gradient is taken through the call."""
    a, out, lse, device = _arguments(query, kv_cache, table, lens, scale, q_start, max_query, prefix_table,
                                     prefix_lens, prefix_rows, k_scale, v_scale, scores, decay, out, lse)
    address = ctypes.addressof(a)
    need = int((ekv_hip._lib or ekv_hip.load()).ekv_prefix_attention_workspace(address))
    workspace = _workspace("workspace", workspace, need, device)
    ekv_hip.call("ekv_prefix_attention", address, workspace.data_ptr(), workspace.numel(),
                 ekv_hip.stream_handle(stream))
    return out, lse
