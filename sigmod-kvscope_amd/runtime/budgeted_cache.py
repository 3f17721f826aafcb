"""One layer's KV cache under a token budget: attention, the weight each cached token accumulates, and the eviction of
the tokens that accumulated least, run together as a serving loop runs them.

Every row owns the pages of ``budget + slack`` tokens for good: an eviction packs what stays into the row's first
slots, so the table never changes.  A prompt that all rows share lies in the cache once.

    cache = BudgetedCache(rows, kv_heads, dim, budget=1024, slack=32)
    cache.set_prefix(keys, values)                  # the shared instructions
    cache.append(keys, values, q_start, longest)    # the rows' prompts
    out, lse = cache.attend(query, scale, q_start, longest)
    while True:                                     # a token a row and step
        cache.append(keys, values)
        out, lse = cache.attend(query, scale)
        if cache.full:
            cache.trim()
"""

from __future__ import annotations

import torch

from runtime.eviction import evict_tokens
from runtime.prefix_attention import prefix_attention


class BudgetedCache:
    """``rows`` rows of at most ``budget + slack`` tokens behind a shared prefix of at most ``prefix`` tokens.  ``recent``
    and ``sinks``: the newest and the first tokens that an eviction spares; ``decay``: what a step leaves of the weight
    accumulated before it; ``k_scale`` / ``v_scale``: an fp8 cache's scales."""

    def __init__(self, rows: int, kv_heads: int, dim: int, budget: int, slack: int = 64, *, prefix: int = 0,
                 block: int = 16, dtype: torch.dtype = torch.bfloat16, recent: int = 32, sinks: int = 4,
                 decay: float = 1.0, k_scale: float = 1.0, v_scale: float = 1.0, device="cuda"):
        if rows < 1 or budget < 1 or slack < 1 or prefix < 0 or block < 1:
            raise ValueError(f"{rows} rows of a budget of {budget} and {slack} tokens, a prefix of {prefix}, blocks of {block}")
        width, shared = -(-(budget + slack) // block), -(-prefix // block)
        pages = 1 + rows * width + shared
        self.capacity, self.budget, self.recent, self.sinks, self.decay = budget + slack, budget, recent, sinks, decay
        self.block, self.k_scale, self.v_scale = block, k_scale, v_scale
        self.kv = torch.zeros(pages, 2, block, kv_heads, dim, dtype=dtype, device=device)
        ids = torch.arange(1, pages, dtype=torch.int32, device=device)
        self.table = ids[: rows * width].view(rows, width)
        self.prefix_table = ids[rows * width:].view(1, shared) if shared else None
        self.prefix_len = torch.zeros(1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=device)
        self.seen = torch.zeros(rows, dtype=torch.int32, device=device)  # the position of a row's next token
        # a row more than there are, and page 0, take the tokens that an append gives to no row
        slots = (rows + 1, kv_heads, width * block)
        self._all_scores = torch.zeros(slots, dtype=torch.float32, device=device)
        self._all_positions = torch.full(slots, -1, dtype=torch.int32, device=device)
        self.scores, self.positions = self._all_scores[:rows], self._all_positions[:rows]
        self._other_lens = torch.zeros_like(self.lens)
        self.longest = 0  # no row has more tokens (the device alone knows each row's)

    @property
    def full(self) -> bool:
        """Whether a row may have no slot left for another token."""
        return self.longest >= self.capacity

    def _check(self, keys: torch.Tensor, values: torch.Tensor) -> None:
        tail = self.kv.shape[3:]
        if keys.ndim != 3 or keys.shape[1:] != tail or values.shape != keys.shape:
            raise ValueError(f"keys and values must be [tokens, {tail[0]}, {tail[1]}], got {tuple(keys.shape)} and {tuple(values.shape)}")

    def _write(self, page: torch.Tensor, slot: torch.Tensor, keys: torch.Tensor, values: torch.Tensor) -> None:
        raw = self.kv.view(torch.uint8) if self.kv.dtype == torch.float8_e4m3fn else self.kv
        for part, rows in ((0, keys), (1, values)):
            rows = rows.to(self.kv.dtype)
            raw[page, part, slot % self.block] = rows.view(torch.uint8) if raw is not self.kv else rows

    def set_prefix(self, keys: torch.Tensor, values: torch.Tensor) -> None:
        """The prefix that every row shares: keys and values ``[tokens, kv_heads, dim]`` (already over an fp8 cache's scales)."""
        self._check(keys, values)
        n = keys.shape[0]
        if self.prefix_table is None or n > self.prefix_table.shape[1] * self.block:
            raise ValueError(f"no room for a prefix of {n} tokens")
        slot = torch.arange(n, device=self.kv.device)
        self._write(self.prefix_table[0, slot // self.block].long(), slot, keys, values)
        self.prefix_len.fill_(n)

    def append(self, keys: torch.Tensor, values: torch.Tensor, q_start: torch.Tensor | None = None, max_query: int = 1) -> None:
        """Each row's next tokens, ``[tokens, kv_heads, dim]``: row r's from ``q_start[r]`` to ``q_start[r + 1]`` (None: one a
        row), at most ``max_query``.  What passes it, or is no row's (padding before or behind the rows'), is not kept: the
        device alone knows the counts, and no row outgrows its pages whatever they are."""
        self._check(keys, values)
        rows, n, device = self.lens.shape[0], keys.shape[0], self.kv.device
        if q_start is None and n != rows:
            raise ValueError(f"{n} tokens of {rows} rows need q_start")
        if q_start is not None and q_start.shape != (rows + 1,):
            raise ValueError(f"q_start must have shape {(rows + 1,)}, got {tuple(q_start.shape)}")
        if max_query < 1:
            raise ValueError(f"at most {max_query} tokens a row")
        if self.longest + max_query > self.capacity:
            raise ValueError(f"{max_query} more tokens pass the {self.capacity} of a row: trim first")
        token = torch.arange(n, device=device)
        if q_start is None:
            row = into = token
            slot, at, counts = self.lens.long(), self.seen, 1
            page = self.table[row, slot // self.block].long()
        else:
            start = q_start.long().clamp(0, n)
            counts = (start[1:] - start[:-1]).clamp(0, max_query).int()
            row = (torch.searchsorted(start, token, right=True) - 1).clamp(0, rows - 1)
            nth = token - start[row]
            kept = (nth >= 0) & (nth < counts[row])
            slot = torch.where(kept, self.lens[row] + nth, 0)
            at = self.seen[row] + nth.int()
            page = torch.where(kept, self.table[row, slot // self.block].long(), 0)
            into = torch.where(kept, row, rows)
        self._write(page, slot, keys, values)
        self._all_scores[into, :, slot] = 0.0
        self._all_positions[into, :, slot] = at[:, None]
        self.lens += counts
        self.seen += counts
        self.longest += max_query

    def attend(self, query: torch.Tensor, scale: float, q_start: torch.Tensor | None = None, max_query: int = 1):
        """``(out, lse)`` of the newest tokens' queries ``[tokens, q_heads, dim]``; the own tokens' scores grow by the weight
        they received."""
        shared = self.prefix_table is not None
        return prefix_attention(
            query, self.kv, self.table, self.lens, scale, q_start=q_start, max_query=max_query,
            prefix_table=self.prefix_table, prefix_lens=self.prefix_len if shared else None, k_scale=self.k_scale,
            v_scale=self.v_scale, scores=self.scores, decay=self.decay)

    def trim(self) -> None:
        """Back to the budget: the tokens that received least are gone."""
        evict_tokens(self.kv, self.table, self.lens, self.scores, self.positions, self.budget, self.seen, recent=self.recent,
                     sinks=self.sinks, new_lens=self._other_lens, new_scores=self.scores, new_positions=self.positions)
        self.lens, self._other_lens = self._other_lens, self.lens
        self.longest = min(self.longest, self.budget)
