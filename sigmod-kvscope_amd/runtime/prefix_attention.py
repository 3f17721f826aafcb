"""Attention over the paged cache for a batch whose rows share prefixes, and the running attention weight of
every cached token.

Requests of a service begin with the same instructions; their keys and values are in the cache once, in
pages every request of the group points to.  Attention that walks each request's own table reads those
pages once per request.  Here a group's queries read them together, once per tile of query rows, on the
matrix cores, and the result joins the attention over each row's own pages through the logarithms of
their sums.  (Rows of long prompt chunks, which fill tiles by themselves, and prefixes too short to be
worth the joining are walked row by row.)

With ``scores`` the call also adds to every own token the weight it received, the running statistic
that ``runtime.eviction.evict_tokens`` ranks tokens by.
"""

from __future__ import annotations

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


_pack = ekv_hip.packer(ekv_hip.Attention)
_INT, _FLOAT = torch.int32, torch.float32


def _sound(device: int, ints, *rows) -> bool:
    """Whether int32 ``(tensor or None, shape)`` pairs and ``(tensor or None, type, shape)`` triples are what the kernels
    read: the usual call's one look at each (``check_tensors`` finds the words for one that is not)."""
    for t, shape in ints:
        if t is not None and not (type(t) is torch.Tensor and t.dtype is _INT and t.shape == shape
                                  and t.get_device() == device and t.stride(-1) == 1):
            return False
    for t, kind, shape in rows:
        if t is not None and not (type(t) is torch.Tensor and t.dtype is kind and t.shape == shape
                                  and t.get_device() == device and t.stride(-1) == 1):
            return False
    return device >= 0


def _arguments(query, kv_cache, table, lens, scale, q_start, max_query, prefix_table, prefix_lens, prefix_rows,
               k_scale, v_scale, scores, decay, out, lse):
    pages, block, kv_heads, dim = _cache_shape(kv_cache)
    if not isinstance(query, torch.Tensor) or query.ndim != 3 or query.shape[2] != dim:
        raise ValueError(f"query must be a [tokens, heads, {dim}] tensor")
    if not isinstance(table, torch.Tensor) or table.ndim != 2:
        raise ValueError("the block table must be a [rows, width] tensor")
    q_shape = tokens, q_heads, _ = query.shape
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
    dtype, device = query.dtype, query.device
    if not (dtype in _QUERY_TYPES and query.stride(2) == 1 and query.is_cuda and _sound(
            query.get_device(),
            ((table, (rows, width)), (lens, (rows,)), (q_start, (rows + 1,)), (prefix_table, (groups, prefix_width)),
             (prefix_lens, (groups,)), (prefix_rows, (groups + 1,))),
            (kv_cache, kv_cache.dtype, kv_cache.shape), (out, dtype, q_shape), (lse, _FLOAT, (tokens, q_heads)))):
        device = check_tensors(
            ("query", query, _QUERY_TYPES, (tokens, q_heads, dim)),
            ("kv_cache", kv_cache, kv_cache.dtype, kv_cache.shape),
            ("table", table, _INT, (rows, width)), ("lens", lens, _INT, (rows,)),
            ("q_start", q_start, _INT, (rows + 1,)),
            ("prefix_table", prefix_table, _INT, (groups, prefix_width)),
            ("prefix_lens", prefix_lens, _INT, (groups,)),
            ("prefix_rows", prefix_rows, _INT, (groups + 1,)),
            ("out", out, dtype, query.shape), ("lse", lse, _FLOAT, (tokens, q_heads)))
    at_scores = score_row = score_head = 0
    if scores is not None:
        if not isinstance(scores, torch.Tensor) or scores.ndim != 3 or scores.shape[:2] != (rows, kv_heads) \
                or scores.shape[2] < width * block:
            raise ValueError(f"scores must be a [{rows}, {kv_heads}, {width * block} or more] tensor")
        if check_tensors(("scores", scores, _FLOAT, scores.shape)) != device:
            raise ValueError(f"scores must be on {device}")
        at_scores, score_row, score_head = scores.data_ptr(), scores.stride(0), scores.stride(1)
    if out is None:
        out = torch.empty(q_shape, dtype=dtype, device=device)
    if lse is None:
        lse = torch.empty(tokens, q_heads, dtype=_FLOAT, device=device)
    elif not lse.is_contiguous():
        raise ValueError("lse must be contiguous")
    q_token, q_head, _ = query.stride()
    kv_block, kv_part, kv_pos, kv_head, _ = kv_cache.stride()
    o_token, o_head, _ = out.stride()
    keys = kv_cache.data_ptr()
    values = keys + kv_part * kv_cache.element_size() if keys else 0
    at_prefix = at_prefix_lens = at_prefix_rows = prefix_stride = 0
    if groups and prefix_width:
        at_prefix, prefix_stride, at_prefix_lens = prefix_table.data_ptr(), prefix_table.stride(0), prefix_lens.data_ptr()
        if prefix_rows is not None:
            at_prefix_rows = prefix_rows.data_ptr()
    else:
        groups = prefix_width = 0
    return _pack(
        query.data_ptr(), q_token, q_head, keys, values, kv_block, kv_pos, kv_head, pages, table.data_ptr(),
        table.stride(0), lens.data_ptr(), 0 if q_start is None else q_start.data_ptr(), at_prefix, prefix_stride,
        at_prefix_lens, at_prefix_rows, at_scores, score_row, score_head, out.data_ptr(), o_token, o_head,
        lse.data_ptr(), ekv_hip.dtype_code(dtype), ekv_hip.dtype_code(kv_cache.dtype), rows, width,
        groups, prefix_width, tokens, max_query, q_heads, kv_heads, dim, block, scale, k_scale, v_scale,
        decay), out, lse, device


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
    every row).  The work is laid out by the tables' widths, the lengths being the device's: tables as wide
    as their longest rows are the fastest.

    ``scores`` float32 ``[rows, kv_heads, slots]``: slot j of each row's tokens becomes ``decay * scores``
    plus the weight its key received from this call's queries.  Types, head dims and limits as
    ``ekv_prefix_attention`` documents them; ``k_scale`` / ``v_scale`` are an fp8 cache's scales.
    ``workspace``: a uint8 device tensor that the call may overwrite (one is allocated if none is given;
    under graph capture it then belongs to the graph's pool).  ``stream``: the call launches and allocates as
    under ``torch.cuda.stream(stream)``; the caller orders it after the work that makes its inputs.  No gradient
    is taken through the call."""
    with ekv_hip.on_stream(stream, query):
        arguments, out, lse, device = _arguments(query, kv_cache, table, lens, scale, q_start, max_query, prefix_table,
                                                 prefix_lens, prefix_rows, k_scale, v_scale, scores, decay, out, lse)
        lib = ekv_hip._lib or ekv_hip.load()
        need = lib.ekv_prefix_attention_workspace(arguments)
        if workspace is None:
            workspace = torch.empty(need or 1, dtype=torch.uint8, device=device)
        else:
            workspace = _workspace("workspace", workspace, need, device)
        status = lib.ekv_prefix_attention(arguments, workspace.data_ptr(), workspace.numel(),
                                          ekv_hip.stream_handle(stream))
    if status:
        ekv_hip.check(status, "ekv_prefix_attention")
    return out, lse
