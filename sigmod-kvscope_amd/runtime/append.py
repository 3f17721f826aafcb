"""A batch's new tokens on their way into a paged cache: keys normed, rotated and, for an fp8 cache, quantised, values
beside them, and the queries normed and rotated for the attention that follows, in one pass.

In a cache whose rows let tokens go (``runtime.eviction.evict_tokens``) a slot is no position: a row's next slot is its
length, its next position the count of tokens it has ever had.  ``append_tokens`` takes both, and starts the running
score and the recorded position of every new slot.
"""

from __future__ import annotations

import torch

import ekv_hip
from observe.allocation import check_tensors
from runtime.prefix_attention import _cache_shape
from runtime.rotary import _heads, _turns, _weights

_pack = ekv_hip.packer(ekv_hip.Append)
_INT, _FLOAT = torch.int32, torch.float32


def append_tokens(
    kv_cache: torch.Tensor,
    table: torch.Tensor,
    lens: torch.Tensor,
    keys: torch.Tensor,
    values: torch.Tensor,
    *,
    q_start: torch.Tensor | None = None,
    max_query: int = 1,
    query: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    frequencies: torch.Tensor | None = None,
    axes: torch.Tensor | None = None,
    adjacent: bool = False,
    rotary_scale: float = 1.0,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    weight_offset: float = 0.0,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
    saturate: bool = True,
    seen: torch.Tensor | None = None,
    first: torch.Tensor | None = None,
    scores: torch.Tensor | None = None,
    slot_positions: torch.Tensor | None = None,
    advance: bool = False,
    q_out: torch.Tensor | None = None,
    stream=None,
) -> torch.Tensor | None:
    """Write the new tokens' ``keys`` and ``values [tokens, kv_heads, dim]`` into their rows' pages; returns the queries,
    normed and rotated (None without ``query [tokens, q_heads, dim]``).

    ``kv_cache [pages, 2, block, kv_heads, dim]`` is written in place through ``table`` int32 ``[rows, width]`` (pages no
    other row uses).  Row r's new tokens are ``q_start[r] .. q_start[r + 1]`` (None: one a row), at most ``max_query``,
    and the last of its ``lens[r]`` tokens, as ``prefix_attention`` takes them afterwards; with ``advance`` they come
    behind the ``lens[r]`` that it has, and the call adds them to ``lens`` (and ``seen``).  A token whose slot is outside
    the row's table, or behind an entry that is no page, is not written.  Tokens of no row write nothing, and their
    queries come back 0.

    Rotation and norms as ``rotate_heads`` has them, before the keys are divided by ``k_scale`` and the values by
    ``v_scale``.  Without ``positions`` a token's is its index in the row, counted by ``seen`` int32 ``[rows]`` (the
    position of the row's next token, kept like ``lens``; None: the slot), plus ``first`` int32 ``[rows]`` (such as the
    length of a prefix; an expanded tensor of one element serves).  An fp8 cache holds what passes +-448 as that with
    ``saturate``, as NaN without.

    ``scores`` float32 and ``slot_positions`` int32 ``[rows, kv_heads, slots]``: 0 and the token's index (without
    ``first``) at each new slot, for every KV head.  ``q_out`` may be ``query`` itself and overlaps nothing else.  Types
    and limits as ``ekv_append_tokens`` documents them.  ``stream``: the call launches and allocates as under
    ``torch.cuda.stream(stream)``; the caller orders it after the work that makes its inputs.  No gradient is taken
    through the call."""
    pages, block, kv_heads, dim = _cache_shape(kv_cache)
    if not isinstance(table, torch.Tensor) or table.ndim != 2:
        raise ValueError("the block table must be a [rows, width] tensor")
    rows, width = table.shape
    tokens, heads, _ = _heads("keys", keys, None, dim, None)
    if heads != kv_heads:
        raise ValueError(f"keys must be a [tokens, {kv_heads}, {dim}] tensor, got {tuple(keys.shape)}")
    dtype, q_heads = keys.dtype, 0
    if kv_cache.dtype != dtype and kv_cache.dtype != torch.float8_e4m3fn:
        raise ValueError(f"keys of {dtype} for a cache of {kv_cache.dtype}")
    if query is not None:
        q_heads = _heads("query", query, tokens, dim, dtype)[1]
    elif q_out is not None or q_weight is not None:
        raise ValueError("q_out and q_weight need a query")
    if frequencies is None and positions is not None:
        raise ValueError("positions need frequencies")
    if width == 0:  # no rows to be contiguous: an empty tensor's strides may be anything
        table = table.new_empty(table.shape)
    if tokens == 0:
        if values.shape != keys.shape or values.dtype != dtype:
            raise ValueError(f"values must be {dtype} of shape {tuple(keys.shape)}")
        keys, values = keys.new_empty(keys.shape), values.new_empty(values.shape)
        query = None if query is None else query.new_empty(query.shape)
    q_shape = None if query is None else query.shape
    device = check_tensors(
        ("kv_cache", kv_cache, kv_cache.dtype, kv_cache.shape), ("keys", keys, dtype, keys.shape),
        ("values", values, dtype, keys.shape), ("query", query, dtype, q_shape), ("q_out", q_out, dtype, q_shape),
        ("table", table, _INT, (rows, width)), ("lens", lens, _INT, (rows,)), ("q_start", q_start, _INT, (rows + 1,)),
        ("seen", seen, _INT, (rows,)))
    at, stride, count, turning, axis, pairs = _turns(tokens, dim, positions, frequencies, axes, device)
    if count == 1 and axes is not None and positions is None:
        raise ValueError("axes need positions")
    qw, kw, qw_stride, kw_stride, w_type = _weights(q_weight, q_heads, k_weight, kv_heads, dim, dtype, device)
    at_first = first_stride = 0
    if first is not None:
        if not isinstance(first, torch.Tensor) or first.shape != (rows,) or first.dtype != _INT or first.device != device:
            raise ValueError(f"first must be an int32 [{rows}] tensor on {device}")
        at_first, first_stride = first.data_ptr(), first.stride(0)
    kept = []
    for name, t, kind in (("scores", scores, _FLOAT), ("slot_positions", slot_positions, _INT)):
        if t is None:
            kept += [0, 0, 0]
            continue
        if not isinstance(t, torch.Tensor) or t.ndim != 3 or t.shape[:2] != (rows, kv_heads) or t.shape[2] < width * block:
            raise ValueError(f"{name} must be a [{rows}, {kv_heads}, {width * block} or more] tensor")
        if check_tensors((name, t, kind, t.shape)) != device:
            raise ValueError(f"{name} must be on {device}")
        kept += [t.data_ptr(), t.stride(0), t.stride(1)]
    with ekv_hip.beside(stream, kv_cache):
        if query is None:
            queries = queries_out = (0, 0, 0)
        else:
            if q_out is None:
                q_out = torch.empty(q_shape, dtype=dtype, device=device)
            queries = (query.data_ptr(), *query.stride()[:2])
            queries_out = (q_out.data_ptr(), *q_out.stride()[:2])
        kv_block, kv_part, kv_pos, kv_head, _ = kv_cache.stride()
        cache = kv_cache.data_ptr()
        arguments = _pack(
            *queries, keys.data_ptr(), values.data_ptr(), *keys.stride()[:2], *values.stride()[:2], *queries_out, cache,
            cache + kv_part * kv_cache.element_size() if cache else 0, kv_block, kv_pos, kv_head, pages, table.data_ptr(),
            table.stride(0), lens.data_ptr(), 0 if seen is None else seen.data_ptr(), at_first, first_stride,
            0 if q_start is None else q_start.data_ptr(), at, stride, turning, axis, qw, kw, qw_stride, kw_stride, *kept,
            ekv_hip.dtype_code(dtype), w_type, ekv_hip.dtype_code(kv_cache.dtype), rows, width, tokens, max_query, q_heads,
            kv_heads, dim, block, pairs, count, bool(adjacent), bool(advance), bool(saturate), rotary_scale, eps,
            weight_offset, k_scale, v_scale, 0)
        status = (ekv_hip._lib or ekv_hip.load()).ekv_append_tokens(arguments, ekv_hip.stream_handle(stream))
    if status:
        ekv_hip.check(status, "ekv_append_tokens")
    return q_out
