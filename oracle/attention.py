"""The definition of attention over a paged cache with shared prefixes, of the running weights and of
token eviction, in float64 NumPy, one query row and one token at a time."""

from __future__ import annotations

import numpy as np


def own_keys(cache: np.ndarray, pages: np.ndarray, n: int) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """Keys, values ``[n, kv_heads, dim]`` of the first n slots behind ``pages``, and which have a page."""
    block = cache.shape[2]
    there = np.zeros(n, dtype=bool)
    keys = np.zeros((n, *cache.shape[3:]))
    values = np.zeros_like(keys)
    for j in range(n):
        page = int(pages[j // block])
        if 0 <= page < cache.shape[0]:
            there[j] = True
            keys[j], values[j] = cache[page, 0, j % block], cache[page, 1, j % block]
    return keys, values, there


def attend(query, cache, table, lens, scale, q_start=None, max_query=1, prefix_table=None, prefix_lens=None,
           prefix_rows=None, k_scale=1.0, v_scale=1.0, scores=None, decay=1.0) -> dict:
    """``out``, ``lse`` and (with ``scores``) the new ``scores``; and for error bounds ``weighed`` (the output of
    the values' magnitudes), ``reach`` (the largest sum of |scale * q * k| over a query's keys) and ``keys``
    (how many it sees)."""
    tokens, q_heads, dim = query.shape
    rows, heads = table.shape[0], cache.shape[3]
    group = q_heads // heads
    start = np.arange(rows + 1) if q_start is None else q_start
    out, weighed = np.zeros((tokens, q_heads, dim)), np.zeros((tokens, q_heads, dim))
    lse = np.full((tokens, q_heads), -np.inf)
    reach, seen = np.zeros((tokens, q_heads)), np.zeros((tokens, q_heads))
    new = None if scores is None else scores.astype(np.float64).copy()
    for r in range(rows):
        n, t = int(lens[r]), int(start[r + 1] - start[r])
        keys, values, there = own_keys(cache, table[r], n)
        if new is not None:
            new[r, :, :n] *= decay
        shared = None
        if prefix_table is not None:
            borders = [0, rows] if prefix_rows is None else prefix_rows
            for g in range(len(prefix_lens)):
                if borders[g] <= r < borders[g + 1]:
                    shared = own_keys(cache, prefix_table[g], int(prefix_lens[g]))
        for i in range(min(t, max_query)):
            token = int(start[r]) + i
            m = min(max(n - t + i + 1, 0), n)
            k, v, ok = keys[:m], values[:m], there[:m]
            p = 0
            if shared is not None:
                p = len(shared[2])
                k, v, ok = (np.concatenate([a, b]) for a, b in zip(shared, (k, v, ok)))
            for hq in range(q_heads):
                h = hq // group
                terms = query[token, hq] * k[:, h] * (scale * k_scale)
                s = np.where(ok, terms.sum(axis=1), -np.inf)
                if not np.any(s > -np.inf):
                    continue
                top = s.max()
                w = np.exp(s - top)
                lse[token, hq] = top + np.log(w.sum())
                w /= w.sum()
                out[token, hq] = v_scale * (w[ok, None] * v[ok, h]).sum(axis=0)
                weighed[token, hq] = abs(v_scale) * (w[ok, None] * np.abs(v[ok, h])).sum(axis=0)
                reach[token, hq], seen[token, hq] = np.abs(terms[ok]).sum(axis=1).max(), ok.sum()
                if new is not None:
                    new[r, h, :m] += np.where(ok, w, 0.0)[p:]
    return {"out": out, "lse": lse, "scores": new, "weighed": weighed, "reach": reach, "keys": seen}


def evict(cache, table, lens, scores, positions, budget, seen, recent=0, sinks=0) -> dict:
    """The cache, scores, positions and lengths after an eviction."""
    rows, heads, capacity = scores.shape
    block = cache.shape[2]
    cache = cache.copy()
    new_scores, new_positions = np.zeros_like(scores), np.full_like(positions, -1)
    new_lens = np.zeros(rows, dtype=np.int32)

    def place(r, j):
        page = int(table[r, j // block])
        return (page, j % block) if 0 <= page < cache.shape[0] else None

    for r in range(rows):
        n = int(lens[r])
        b = new_lens[r] = min(n, max(int(budget[r]), 0))
        for h in range(heads):
            def rank(j):
                x = float(scores[r, h, j])
                p = int(positions[r, h, j])
                safe = p < sinks or p >= int(seen[r]) - recent
                return (not safe, np.inf if x != x else -x, j)

            best = sorted(sorted(range(n), key=rank)[:b])
            late = [j for j in best if j >= b]
            freed = [j for j in range(b) if j not in set(best)]
            source = list(range(b))
            for a, z in zip(late, freed):
                source[z] = a
                x, y = place(r, a), place(r, z)
                if x and y:
                    cache[y[0], :, y[1], h] = cache[x[0], :, x[1], h]
            new_scores[r, h, :b], new_positions[r, h, :b] = scores[r, h, source], positions[r, h, source]
    return {"cache": cache, "scores": new_scores, "positions": new_positions, "lens": new_lens}
