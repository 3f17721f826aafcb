"""The definition of head norms, of the rotation of positions and of appending to a paged cache, in float64 NumPy, one
token at a time."""

from __future__ import annotations

import numpy as np


def rotate(x, weight, eps, offset, positions, frequencies, axes=None, adjacent=False, scale=1.0):
    """One token's heads ``[heads, dim]`` normed (``weight`` None: not) and rotated by ``positions [axes]``; and for error
    bounds the magnitude that each element's terms sum to.  A pair of an axis that is not there turns by position 0."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * (offset + np.asarray(weight, np.float64))
    y, reach = x.copy(), np.abs(x)
    pairs = 0 if frequencies is None else len(frequencies)
    if pairs:
        axis = np.zeros(pairs, int) if axes is None else np.asarray(axes)
        there = (axis >= 0) & (axis < len(positions))
        angle = np.where(there, np.asarray(positions, np.float64)[np.where(there, axis, 0)], 0.0) * frequencies
        p = np.arange(pairs)
        a, b = (2 * p, 2 * p + 1) if adjacent else (p, p + pairs)
        y[:, a] = scale * (x[:, a] * np.cos(angle) - x[:, b] * np.sin(angle))
        y[:, b] = scale * (x[:, a] * np.sin(angle) + x[:, b] * np.cos(angle))
        reach[:, a] = reach[:, b] = abs(scale) * (np.abs(x[:, a]) + np.abs(x[:, b]))
    return y, reach


def append(cache, table, lens, keys, values, q_start=None, max_query=1, query=None, positions=None, frequencies=None,
           axes=None, adjacent=False, rotary_scale=1.0, q_weight=None, k_weight=None, eps=1e-6, weight_offset=0.0,
           k_scale=1.0, v_scale=1.0, seen=None, first=None, scores=None, slot_positions=None, advance=False) -> dict:
    """The cache (unrounded), the queries, scores, slot positions, lengths and counts after an append; ``wrote`` marks the
    cache's new elements, ``reach`` and ``query_reach`` are the magnitudes of their terms."""
    rows, block, capacity = table.shape[0], cache.shape[2], table.shape[1] * cache.shape[2]
    tokens = keys.shape[0]
    start = np.arange(rows + 1) if q_start is None else np.clip(q_start, 0, tokens)
    out = {"cache": cache.astype(np.float64), "reach": np.zeros(cache.shape), "wrote": np.zeros(cache.shape, bool),
           "lens": np.array(lens), "query": None if query is None else np.zeros(query.shape),
           "query_reach": None if query is None else np.zeros(query.shape),
           "seen": None if seen is None else np.array(seen), "scores": None if scores is None else scores.copy(),
           "slot_positions": None if slot_positions is None else slot_positions.copy()}
    turn = dict(frequencies=frequencies, axes=axes, adjacent=adjacent, scale=rotary_scale)
    for r in range(rows):
        t = int(start[r + 1] - start[r])
        n = min(max(int(lens[r]), 0), capacity)
        back = 0 if advance else t
        for i in range(min(t, max_query)):
            token, slot = int(start[r]) + i, n - back + i
            index = slot if seen is None else int(seen[r]) - back + i
            where = [index + (0 if first is None else int(first[r]))] if positions is None else positions[:, token]
            if query is not None:
                out["query"][token], out["query_reach"][token] = rotate(query[token], q_weight, eps, weight_offset, where, **turn)
            if not 0 <= slot < capacity:
                continue
            if scores is not None:
                out["scores"][r, :, slot] = 0.0
            if slot_positions is not None:
                out["slot_positions"][r, :, slot] = index
            page, at = int(table[r, slot // block]), slot % block
            if not 0 <= page < cache.shape[0]:
                continue
            key, reach = rotate(keys[token], k_weight, eps, weight_offset, where, **turn)
            out["cache"][page, 0, at], out["reach"][page, 0, at] = key / k_scale, reach / k_scale
            out["cache"][page, 1, at] = values[token] / v_scale
            out["reach"][page, 1, at] = np.abs(values[token]) / v_scale
            out["wrote"][page, :, at] = True
        kept = min(t, max_query)
        if advance and kept > 0:
            out["lens"][r] = n + min(kept, capacity - n)
            if seen is not None:
                out["seen"][r] += kept
    return out
