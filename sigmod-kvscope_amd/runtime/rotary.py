"""Rotary positions and the norms of query and key heads, in one pass over what the projection leaves.

A pair of a head's elements turns by its token's position times the pair's frequency.  Positions may have several axes
(time, height and width of an image's or a video's patches): ``axes`` then names the axis of each pair.  Where a model
norms its query and key heads first, the same pass does it.  ``runtime.append.append_tokens`` does the same on the
way into a paged cache.
"""

from __future__ import annotations

import torch

import ekv_hip
from observe.allocation import check_tensors

_HEAD_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_pack = ekv_hip.packer(ekv_hip.Rotation)
_INT = torch.int32


def rotary_frequencies(pairs: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """``base ** -(p / pairs)`` radians a position for pair p, float64 ``[pairs]``."""
    if pairs < 1 or not base > 0:
        raise ValueError(f"{pairs} pairs of base {base}")
    return torch.pow(float(base), -torch.arange(pairs, dtype=torch.float64) / pairs).to(device)


def section_axes(*pairs: int, interleaved: bool = False, device="cuda") -> torch.Tensor:
    """The axis of each pair, int32: ``pairs[a]`` of them belong to axis a.  In a run each, or ``interleaved``: axis a
    takes pairs a, a + n, a + 2 n ... of n axes until it has its own, the first axis all that are left."""
    n, total = len(pairs), sum(pairs)
    if not n or min(pairs) < 0:
        raise ValueError(f"sections of {pairs} pairs")
    if interleaved:
        axis = [0] * total
        for a in range(1, n):
            if pairs[a] and a + n * (pairs[a] - 1) >= total:
                raise ValueError(f"{pairs[a]} pairs of axis {a} do not fit every {n}th of {total}")
            axis[a:a + n * pairs[a]:n] = [a] * pairs[a]
    else:
        axis = [a for a, count in enumerate(pairs) for _ in range(count)]
    return torch.tensor(axis, dtype=_INT, device=device)


def _heads(name: str, t, tokens: int | None, dim: int | None, dtype) -> tuple[int, int, int]:
    """(tokens, heads, dim) of a ``[tokens, heads, dim]`` tensor whose other sizes and type are known."""
    if not isinstance(t, torch.Tensor) or t.ndim != 3:
        raise ValueError(f"{name} must be a [tokens, heads, dim] tensor")
    shape = t.shape
    if (tokens is not None and shape[0] != tokens) or (dim is not None and shape[2] != dim):
        raise ValueError(f"{name} must be a [{tokens}, heads, {dim}] tensor, got {tuple(shape)}")
    if t.dtype not in _HEAD_TYPES or (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{name} must be {_HEAD_TYPES if dtype is None else dtype}, got {t.dtype}")
    return shape


def _turns(tokens: int, dim: int, positions, frequencies, axes, device) -> tuple[int, ...]:
    """The fields (positions, stride, axes of them, frequencies, axes, pairs)."""
    if frequencies is None:
        if axes is not None:
            raise ValueError("axes need frequencies")
        return 0, 0, 1, 0, 0, 0
    if not isinstance(frequencies, torch.Tensor) or frequencies.ndim != 1:
        raise ValueError("frequencies must be a [pairs] tensor")
    pairs = frequencies.shape[0]
    if 2 * pairs > dim:
        raise ValueError(f"{pairs} pairs of heads of {dim}")
    at = stride = 0
    count = 1
    if positions is not None:
        if not isinstance(positions, torch.Tensor) or positions.ndim not in (1, 2) or positions.shape[-1] != tokens:
            raise ValueError(f"positions must be a [{tokens}] or [axes, {tokens}] tensor")
        if positions.ndim == 2:
            count, stride = positions.shape[0], positions.stride(0)
        at = positions.data_ptr()
    if check_tensors(("frequencies", frequencies, torch.float64, (pairs,)), ("axes", axes, _INT, (pairs,)),
                     ("positions", positions if tokens else None, _INT, None if positions is None else positions.shape)) != device:
        raise ValueError(f"frequencies must be on {device}")
    if axes is None and count > 1:
        raise ValueError(f"positions of {count} axes need axes")
    return at, stride, count, frequencies.data_ptr(), 0 if axes is None else axes.data_ptr(), pairs


def _weights(q_weight, q_heads: int, k_weight, kv_heads: int, dim: int, dtype, device) -> tuple[int, int, int, int, int]:
    """The fields (q weight, k weight, their strides, type)."""
    kind, fields = None, []
    for name, w, heads in (("q_weight", q_weight, q_heads), ("k_weight", k_weight, kv_heads)):
        if w is None:
            fields.append((0, 0))
            continue
        if not isinstance(w, torch.Tensor) or w.shape not in ((dim,), (heads, dim)):
            raise ValueError(f"{name} must be a [{dim}] or [{heads}, {dim}] tensor")
        if w.dtype != dtype and w.dtype != torch.float32:
            raise ValueError(f"{name} must be {dtype} or float32, got {w.dtype}")
        if kind is not None and w.dtype != kind:
            raise ValueError(f"k_weight must be {kind} as q_weight is, got {w.dtype}")
        kind = w.dtype
        if check_tensors((name, w, kind, w.shape)) != device:
            raise ValueError(f"{name} must be on {device}")
        fields.append((w.data_ptr(), w.stride(0) if w.ndim == 2 and heads > 1 else 0))
    return fields[0][0], fields[1][0], fields[0][1], fields[1][1], ekv_hip.dtype_code(dtype if kind is None else kind)


def rotate_heads(
    query: torch.Tensor,
    key: torch.Tensor | None,
    positions: torch.Tensor | None,
    frequencies: torch.Tensor | None,
    *,
    axes: torch.Tensor | None = None,
    adjacent: bool = False,
    rotary_scale: float = 1.0,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    weight_offset: float = 0.0,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
    stream=None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``query [tokens, q_heads, dim]`` and ``key [tokens, kv_heads, dim]`` (None: none), normed and rotated.

    ``positions`` int32 ``[tokens]`` or ``[axes, tokens]``; ``frequencies`` float64 ``[pairs]``, radians a position
    (``rotary_frequencies`` makes the usual ones; None: norms alone); ``axes`` int32 ``[pairs]``, the axis of each pair
    (``section_axes``).  Pair p is elements p and p + pairs of a head, or with ``adjacent`` elements 2 p and 2 p + 1;
    those from 2 * pairs on stay as they are.  ``rotary_scale`` multiplies what rotates.

    ``q_weight`` and ``k_weight`` ``[dim]`` or ``[heads, dim]``, of the heads' type or float32: each head is first
    divided by its root mean square (``eps`` added to the mean square) and multiplied by ``weight_offset`` plus its
    weights.  None: that tensor is not normed.

    ``q_out`` and ``k_out`` may be ``query`` and ``key`` themselves and overlap nothing else.  Types, head dims and
    limits as ``ekv_rotate_heads`` documents them.  ``stream``: the call launches and allocates as under
    ``torch.cuda.stream(stream)``; the caller orders it after the work that makes its inputs.  No gradient is taken
    through the call."""
    tokens, q_heads, dim = _heads("query", query, None, None, None)
    dtype, kv_heads = query.dtype, 0
    if key is not None:
        kv_heads = _heads("key", key, tokens, dim, dtype)[1]
    elif k_out is not None or k_weight is not None:
        raise ValueError("k_out and k_weight need a key")
    if frequencies is not None and positions is None:
        raise ValueError("frequencies need positions")
    if tokens == 0:  # no rows to be contiguous: an empty tensor's strides may be anything
        query, key = query.new_empty(query.shape), None if key is None else key.new_empty(key.shape)
    device = check_tensors(("query", query, dtype, query.shape), ("key", key, dtype, None if key is None else key.shape),
                           ("q_out", q_out, dtype, query.shape), ("k_out", k_out, dtype, None if key is None else key.shape))
    at, stride, count, turning, axis, pairs = _turns(tokens, dim, positions, frequencies, axes, device)
    qw, kw, qw_stride, kw_stride, w_type = _weights(q_weight, q_heads, k_weight, kv_heads, dim, dtype, device)
    with ekv_hip.beside(stream, query):
        if q_out is None:
            q_out = torch.empty(query.shape, dtype=dtype, device=device)
        if k_out is None and key is not None:
            k_out = torch.empty(key.shape, dtype=dtype, device=device)
        keys = (0, 0, 0) if key is None else (key.data_ptr(), *key.stride()[:2])
        keys_out = (0, 0, 0) if key is None else (k_out.data_ptr(), *k_out.stride()[:2])
        arguments = _pack(
            query.data_ptr(), *query.stride()[:2], *keys, q_out.data_ptr(), *q_out.stride()[:2], *keys_out, at, stride,
            turning, axis, qw, kw, qw_stride, kw_stride, ekv_hip.dtype_code(dtype), w_type, tokens, q_heads, kv_heads, dim,
            pairs, count, bool(adjacent), rotary_scale, eps, weight_offset)
        status = (ekv_hip._lib or ekv_hip.load()).ekv_rotate_heads(arguments, ekv_hip.stream_handle(stream))
    if status:
        ekv_hip.check(status, "ekv_rotate_heads")
    return q_out, k_out
