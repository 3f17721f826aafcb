"""Eviction of cached tokens by the attention weight they accumulated.

``runtime.prefix_attention.prefix_attention`` keeps a running weight of every cached token.  When a row
outgrows its budget, ``evict_tokens`` keeps the heaviest tokens of each KV head, with the first few (which
attention always returns to) and the newest (which had no time to accumulate) protected, and packs them into
the row's first slots so that its last pages can be freed.  Attention does not depend on the order of the
slots, so only tokens behind the budget move, each into a freed slot.
"""

from __future__ import annotations

import ctypes

import torch

import ekv_hip
from observe.allocation import _workspace, check_tensors
from runtime.prefix_attention import _cache_shape


def eviction_workspace_bytes(rows: int, kv_heads: int, capacity: int) -> int:
    """Device bytes ``evict_tokens`` needs for rows of ``capacity`` slots."""
    return int((ekv_hip._lib or ekv_hip.load()).ekv_evict_tokens_workspace(rows, kv_heads, capacity))


def evict_tokens(
    kv_cache: torch.Tensor,
    table: torch.Tensor,
    lens: torch.Tensor,
    scores: torch.Tensor,
    positions: torch.Tensor,
    budget: int | torch.Tensor,
    seen: torch.Tensor,
    *,
    recent: int = 0,
    sinks: int = 0,
    new_lens: torch.Tensor | None = None,
    new_scores: torch.Tensor | None = None,
    new_positions: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    stream=None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Keep ``budget`` tokens of every row and KV head; returns ``(new_lens, new_scores, new_positions)``.

    ``kv_cache [pages, 2, block, kv_heads, dim]`` is rewritten in place through ``table`` int32
    ``[rows, width]`` (pages no other row uses) for rows of ``lens`` tokens; ``scores`` float32 and
    ``positions`` int32 ``[rows, kv_heads, width * block]`` hold each slot's weight and the position its
    token had in the row; ``budget`` an int or int32 ``[rows]``; ``seen`` int32 ``[rows]`` the position the
    next token will have.  Tokens of a position below ``sinks`` or at ``seen - recent`` and later come first,
    then higher scores, then lower slots; NaN ranks lowest.  The k-th token kept behind the budget moves
    into the k-th freed slot before it.  The new buffers may be the old ones (``scores`` and ``positions``,
    not ``lens``); slots past the new length get score 0 and position -1."""
    pages, block, kv_heads, dim = _cache_shape(kv_cache)
    if not isinstance(table, torch.Tensor) or table.ndim != 2:
        raise ValueError("the block table must be a [rows, width] tensor")
    rows, width = table.shape
    shape = (rows, kv_heads, width * block)
    per_row = budget if isinstance(budget, torch.Tensor) else None
    device = check_tensors(
        ("kv_cache", kv_cache, kv_cache.dtype, kv_cache.shape), ("table", table, torch.int32, (rows, width)),
        ("lens", lens, torch.int32, (rows,)), ("scores", scores, torch.float32, shape),
        ("positions", positions, torch.int32, shape), ("budget", per_row, torch.int32, (rows,)),
        ("seen", seen, torch.int32, (rows,)), ("new_lens", new_lens, torch.int32, (rows,)),
        ("new_scores", new_scores, torch.float32, shape), ("new_positions", new_positions, torch.int32, shape))
    if new_lens is None:
        new_lens = torch.empty(rows, dtype=torch.int32, device=device)
    if new_scores is None:
        new_scores = torch.empty(shape, dtype=torch.float32, device=device)
    if new_positions is None:
        new_positions = torch.empty(shape, dtype=torch.int32, device=device)
    a = ekv_hip.Eviction()
    stride = kv_cache.stride()
    a.keys = kv_cache.data_ptr()
    a.values = a.keys + stride[1] * kv_cache.element_size() if a.keys else 0
    a.kv_stride_block, a.kv_stride_pos, a.kv_stride_head, a.blocks = stride[0], stride[2], stride[3], pages
    a.table, a.table_stride, a.lens, a.seen = table.data_ptr(), table.stride(0), lens.data_ptr(), seen.data_ptr()
    if per_row is None:
        a.fixed_budget = int(budget)
    else:
        a.budget = per_row.data_ptr()
    a.scores, (a.scores_stride_row, a.scores_stride_head, _) = scores.data_ptr(), scores.stride()
    a.positions, (a.positions_stride_row, a.positions_stride_head, _) = positions.data_ptr(), positions.stride()
    a.new_scores, (a.new_scores_stride_row, a.new_scores_stride_head, _) = new_scores.data_ptr(), new_scores.stride()
    a.new_positions, (a.new_positions_stride_row, a.new_positions_stride_head, _) = (new_positions.data_ptr(),
                                                                                     new_positions.stride())
    a.new_lens = new_lens.data_ptr()
    a.kv_dtype = ekv_hip.dtype_code(kv_cache.dtype)
    a.rows, a.kv_heads, a.head_dim, a.width, a.block_size = rows, kv_heads, dim, width, block
    a.recent, a.sinks = int(recent), int(sinks)
    workspace = _workspace("workspace", workspace, eviction_workspace_bytes(rows, kv_heads, width * block), device)
    ekv_hip.call("ekv_evict_tokens", ctypes.addressof(a), workspace.data_ptr(), workspace.numel(),
                 ekv_hip.stream_handle(stream))
    return new_lens, new_scores, new_positions
