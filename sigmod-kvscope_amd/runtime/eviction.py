"""Eviction of cached tokens by the attention weight they accumulated.

``runtime.prefix_attention.prefix_attention`` keeps a running weight of every cached token.  When a row
outgrows its budget, ``evict_tokens`` keeps the heaviest tokens of each KV head, with the first few (which
attention always returns to) and the newest (which had no time to accumulate) protected, and packs them into
the row's first slots so that its last pages can be freed.  Attention does not depend on the order of the
slots, so only tokens behind the budget move, each into a freed slot.
"""

from __future__ import annotations

import torch

import ekv_hip
from observe.allocation import _workspace, check_tensors
from runtime.prefix_attention import _FLOAT, _INT, _cache_shape, _sound

_pack = ekv_hip.packer(ekv_hip.Eviction)


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
    not ``lens``); slots past the new length get score 0 and position -1.  ``stream``: the call launches and
    allocates as under ``torch.cuda.stream(stream)``."""
    pages, block, kv_heads, dim = _cache_shape(kv_cache)
    if not isinstance(table, torch.Tensor) or table.ndim != 2:
        raise ValueError("the block table must be a [rows, width] tensor")
    rows, width = table.shape
    shape = (rows, kv_heads, width * block)
    per_row = budget if isinstance(budget, torch.Tensor) else None
    device = kv_cache.device
    if not (kv_cache.is_cuda and _sound(
            kv_cache.get_device(),
            ((table, (rows, width)), (lens, (rows,)), (positions, shape), (per_row, (rows,)), (seen, (rows,)),
             (new_lens, (rows,)), (new_positions, shape)),
            (kv_cache, kv_cache.dtype, kv_cache.shape), (scores, _FLOAT, shape), (new_scores, _FLOAT, shape))):
        device = check_tensors(
            ("kv_cache", kv_cache, kv_cache.dtype, kv_cache.shape), ("table", table, _INT, (rows, width)),
            ("lens", lens, _INT, (rows,)), ("scores", scores, _FLOAT, shape),
            ("positions", positions, _INT, shape), ("budget", per_row, _INT, (rows,)),
            ("seen", seen, _INT, (rows,)), ("new_lens", new_lens, _INT, (rows,)),
            ("new_scores", new_scores, _FLOAT, shape), ("new_positions", new_positions, _INT, shape))
    with ekv_hip.on_stream(stream, kv_cache):
        if new_lens is None:
            new_lens = torch.empty(rows, dtype=_INT, device=device)
        if new_scores is None:
            new_scores = torch.empty(shape, dtype=_FLOAT, device=device)
        if new_positions is None:
            new_positions = torch.empty(shape, dtype=_INT, device=device)
        kv_block, kv_part, kv_pos, kv_head, _ = kv_cache.stride()
        keys = kv_cache.data_ptr()
        values = keys + kv_part * kv_cache.element_size() if keys else 0
        s_row, s_head, _ = scores.stride()
        p_row, p_head, _ = positions.stride()
        ns_row, ns_head, _ = new_scores.stride()
        np_row, np_head, _ = new_positions.stride()
        arguments = _pack(
            keys, values, kv_block, kv_pos, kv_head, pages, table.data_ptr(), table.stride(0), lens.data_ptr(),
            0 if per_row is None else per_row.data_ptr(), seen.data_ptr(), scores.data_ptr(), s_row, s_head,
            positions.data_ptr(), p_row, p_head, new_scores.data_ptr(), ns_row, ns_head, new_positions.data_ptr(), np_row,
            np_head, new_lens.data_ptr(), ekv_hip.dtype_code(kv_cache.dtype), rows, kv_heads, dim, width, block,
            int(budget) if per_row is None else 0, int(recent), int(sinks), 0)
        lib = ekv_hip._lib or ekv_hip.load()
        need = lib.ekv_evict_tokens_workspace(rows, kv_heads, width * block)
        if workspace is None:
            workspace = torch.empty(need or 1, dtype=torch.uint8, device=device)
        else:
            workspace = _workspace("workspace", workspace, need, device)
        status = lib.ekv_evict_tokens(arguments, workspace.data_ptr(), workspace.numel(), ekv_hip.stream_handle(stream))
    if status:
        ekv_hip.check(status, "ekv_evict_tokens")
    return new_lens, new_scores, new_positions
