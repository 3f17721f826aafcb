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
from runtime.prefix_attention import _cache_shape, _sound
from runtime.rotary import _HEAD_TYPES, _HERE, _NO_WEIGHTS, _look, _output, _turns, _weights

_pack = ekv_hip.packer(ekv_hip.Append)
_INT, _FLOAT = torch.int32, torch.float32
_FP8 = torch.float8_e4m3fn
_Tensor = torch.Tensor
_NONE = (0, 0, 0)


def _slots(name: str, t, kind, rows: int, heads: int, least: int, device: int) -> tuple[int, int, int]:
    """(address, strides of the rows and heads) of a tensor with a value for every slot."""
    if not isinstance(t, _Tensor) or t.ndim != 3 or t.shape[:2] != (rows, heads) or t.shape[2] < least:
        raise ValueError(f"{name} must be a [{rows}, {heads}, {least} or more] tensor")
    row, head, one = t.stride()
    if t.dtype is not kind or one != 1 or t.get_device() != device:
        if check_tensors((name, t, kind, t.shape)).index != device:
            raise ValueError(f"{name} must be on the cache's device, got {t.device}")
    return t.data_ptr(), row, head


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
    behind the ``lens[r]`` that it has, and the call adds them to ``lens`` (and ``seen``; neither shares memory with the
    other or with ``first``; ``prefix_attention`` takes them with this ``max_query`` as its
    ``kept``).  A token whose slot is outside
    the row's table, or behind an entry that is no page, is not written.  Tokens of no row write nothing, and their
    queries come back 0.

    Rotation and norms as ``rotate_heads`` has them, before the keys are divided by ``k_scale`` and the values by
    ``v_scale``.  Without ``positions`` a token's is its index in the row, counted by ``seen`` int32 ``[rows]`` (the
    position of the row's next token, kept like ``lens``; None: the slot), plus ``first`` int32 ``[rows]`` (such as the
    length of a prefix; an expanded tensor of one element serves).  An fp8 cache holds what passes +-448 as that with
    ``saturate``, as NaN without.

    ``scores`` float32 and ``slot_positions`` int32 ``[rows, kv_heads, slots]``: 0 and the token's index (without
    ``first``) at each new slot, for every KV head.  ``q_out`` may be ``query`` itself; its heads overlap
    nothing else, nor each other.  Types and limits as ``ekv_append_tokens`` documents them.  ``stream``: the call launches
    and allocates as under ``torch.cuda.stream(stream)``; the caller orders it after the work that makes its inputs.  No
    gradient is taken through the call."""
    if not isinstance(kv_cache, _Tensor) or kv_cache.ndim != 5:
        _cache_shape(kv_cache)  # refuses it
    pages, _, block, kv_heads, dim = c_shape = kv_cache.shape
    kv_block, kv_part, kv_pos, kv_head, kv_one = kv_cache.stride()
    if c_shape[1] != 2 or kv_one != 1 or block < 1 or kv_heads < 1:
        _cache_shape(kv_cache)
    if not isinstance(table, _Tensor) or table.ndim != 2:
        raise ValueError("the block table must be a [rows, width] tensor")
    rows, width = t_shape = table.shape
    t_row, t_one = table.stride()
    k_shape, dtype, k_device, k_at, k_token, k_head, sound = _look("keys", keys)
    tokens, heads, k_dim = k_shape
    if heads != kv_heads or k_dim != dim:
        raise ValueError(f"keys must be a [tokens, {kv_heads}, {dim}] tensor, got {tuple(k_shape)}")
    kv_dtype, device = kv_cache.dtype, kv_cache.get_device()
    if kv_dtype is not dtype and kv_dtype is not _FP8:
        raise ValueError(f"keys of {dtype} for a cache of {kv_dtype}")
    v_shape, v_type, v_device, v_at, v_token, v_head, v_sound = _look("values", values)
    sound = sound and v_sound and v_shape == k_shape and v_type is dtype and k_device == v_device == device
    q_shape, q_heads, q_at, q_token, q_head = None, 0, 0, 0, 0
    if query is not None:
        q_shape, q_type, q_device, q_at, q_token, q_head, q_sound = _look("query", query)
        q_tokens, q_heads, q_dim = q_shape
        if q_tokens != tokens or q_dim != dim:
            raise ValueError(f"query must be a [{tokens}, heads, {dim}] tensor, got {tuple(q_shape)}")
        sound = sound and q_sound and q_type is dtype and q_device == device
    elif q_out is not None or q_weight is not None:
        raise ValueError("q_out and q_weight need a query")
    if frequencies is None and positions is not None:
        raise ValueError("positions need frequencies")
    if not sound or device < 0 or dtype not in _HEAD_TYPES or table.dtype is not _INT or t_one != 1 \
            or table.get_device() != device or not isinstance(lens, _Tensor) or lens.dtype is not _INT or lens.shape != (rows,) \
            or lens.get_device() != device or lens.stride() != (1,) or ((q_start is not None or seen is not None) and not _sound(
                device, ((q_start, (rows + 1,)), (seen, (rows,))))):
        if width == 0:  # no rows to be contiguous: an empty tensor's strides may be anything
            table = table.new_empty(t_shape)
        if tokens == 0:
            if v_shape != k_shape or v_type != dtype:
                raise ValueError(f"values must be {dtype} of shape {tuple(k_shape)}, got {v_type} of {tuple(v_shape)}")
            keys, values = keys.new_empty(k_shape), values.new_empty(k_shape)
            query = None if query is None else query.new_empty(q_shape)
        check_tensors(
            ("kv_cache", kv_cache, kv_dtype, c_shape), ("keys", keys, _HEAD_TYPES, k_shape),
            ("values", values, dtype, k_shape), ("query", query, dtype, q_shape),
            ("q_out", q_out, dtype, q_shape), ("table", table, _INT, t_shape), ("lens", lens, _INT, (rows,)),
            ("q_start", q_start, _INT, (rows + 1,)), ("seen", seen, _INT, (rows,)))
    at, stride, count, turning, axis, pairs = _turns(tokens, dim, positions, frequencies, axes, device)
    q_weighs, k_weighs, q_step, k_step, w_type = _NO_WEIGHTS if q_weight is None and k_weight is None else \
        _weights(q_weight, q_heads, k_weight, kv_heads, dim, dtype, device)
    at_first = first_stride = 0
    if first is not None:
        if not isinstance(first, _Tensor) or first.shape != (rows,) or first.dtype != _INT or first.get_device() != device:
            raise ValueError(f"first must be an int32 [{rows}] tensor on the cache's device")
        at_first, first_stride = first.data_ptr(), first.stride(0)
    s_at, s_row, s_head = _NONE if scores is None else _slots("scores", scores, _FLOAT, rows, kv_heads, width * block, device)
    p_at, p_row, p_head = _NONE if slot_positions is None else \
        _slots("slot_positions", slot_positions, _INT, rows, kv_heads, width * block, device)
    context, handle = ekv_hip.beside(stream, kv_cache)
    with context or _HERE:
        o_at = o_token = o_head = 0
        if query is not None:
            if q_out is None:
                q_out = torch.empty(tokens, q_heads, dim, dtype=dtype, device=kv_cache.device)
                o_at, o_token, o_head = q_out.data_ptr(), q_heads * dim, dim
            else:
                o_at, o_token, o_head = _output("q_out", q_out, dtype, q_shape, kv_cache)
        cache = kv_cache.data_ptr()
        arguments = _pack(
            q_at, q_token, q_head, k_at, v_at, k_token, k_head, v_token, v_head, o_at, o_token, o_head, cache,
            cache + kv_part * kv_cache.element_size() if cache else 0, kv_block, kv_pos, kv_head, pages, table.data_ptr(),
            t_row, lens.data_ptr(), 0 if seen is None else seen.data_ptr(), at_first, first_stride,
            0 if q_start is None else q_start.data_ptr(), at, stride, turning, axis, q_weighs, k_weighs, q_step, k_step,
            s_at, s_row, s_head, p_at, p_row, p_head, ekv_hip.dtype_code(dtype), w_type, ekv_hip.dtype_code(kv_dtype), rows,
            width, tokens, max_query, q_heads, kv_heads, dim, block, pairs, count, 1 if adjacent else 0, 1 if advance else 0,
            1 if saturate else 0, rotary_scale, eps, weight_offset, k_scale, v_scale, 0)
        status = (ekv_hip._lib or ekv_hip.load()).ekv_append_tokens(arguments, handle)
    if status:
        ekv_hip.check(status, "ekv_append_tokens")
    return q_out
