"""Rotary positions and the norms of query and key heads, in one pass over what the projection leaves.

A pair of a head's elements turns by its token's position times the pair's frequency.  Positions may have several axes
(time, height and width of an image's or a video's patches): ``axes`` then names the axis of each pair.  Where a model
norms its query and key heads first, the same pass does it.  ``runtime.append.append_tokens`` does the same on the
way into a paged cache.
"""

from __future__ import annotations

import contextlib

import torch

import ekv_hip
from observe.allocation import check_tensors

_HEAD_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_pack = ekv_hip.packer(ekv_hip.Rotation)
_INT = torch.int32
_Tensor = torch.Tensor
_STILL = (0, 0, 1, 0, 0, 0)  # no rotation
_NO_WEIGHTS = (0, 0, 0, 0, 0)
_HERE = contextlib.nullcontext()


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


def _look(name: str, t) -> tuple:
    """(shape, type, device, address, strides of the tokens and heads, whether rows are contiguous) of a ``[tokens, heads,
    dim]`` tensor: the usual call's one look at it (``check_tensors`` finds the words for one that is not sound)."""
    if isinstance(t, _Tensor):
        shape = t.shape
        if len(shape) == 3:
            token, head, one = t.stride()
            return shape, t.dtype, t.get_device(), t.data_ptr(), token, head, one == 1 or shape[0] == 0
    raise ValueError(f"{name} must be a [tokens, heads, dim] tensor")


def _output(name: str, t, dtype, shape, like) -> tuple[int, int, int]:
    """(address, strides of the tokens and heads) of a given output, which is of ``like``'s device."""
    o_shape, o_type, o_device, at, token, head, sound = _look(name, t)
    if not sound or o_shape != shape or o_type is not dtype or o_device != like.get_device():
        check_tensors(("the input", like, like.dtype, like.shape), (name, t, dtype, shape))
    return at, token, head


def _turns(tokens: int, dim: int, positions, frequencies, axes, device: int) -> tuple[int, ...]:
    """The fields (positions, their stride and axes, frequencies, axes, pairs)."""
    if frequencies is None:
        if axes is not None or positions is not None:
            raise ValueError("axes and positions need frequencies")
        return _STILL
    if not isinstance(frequencies, _Tensor) or frequencies.ndim != 1:
        raise ValueError("frequencies must be a [pairs] tensor")
    pairs, = frequencies.shape
    if 2 * pairs > dim:
        raise ValueError(f"{pairs} pairs of heads of {dim}")
    at = stride = axis = 0
    count = 1
    sound = frequencies.dtype is torch.float64 and frequencies.get_device() == device and frequencies.stride() == (1,)
    if positions is not None:
        if not isinstance(positions, _Tensor) or positions.ndim not in (1, 2) or positions.shape[-1] != tokens:
            raise ValueError(f"positions must be a [{tokens}] or [axes, {tokens}] tensor")
        steps = positions.stride()
        if len(steps) == 2:
            count, stride = positions.shape[0], steps[0]
        at = positions.data_ptr()
        sound = sound and positions.dtype is _INT and positions.get_device() == device and (steps[-1] == 1 or tokens == 0)
    elif axes is not None:
        raise ValueError("axes need positions")
    if axes is not None:
        axis = axes.data_ptr() if isinstance(axes, _Tensor) else 0
        sound = sound and isinstance(axes, _Tensor) and axes.dtype is _INT and axes.shape == (pairs,) \
            and axes.get_device() == device and axes.stride() == (1,)
    elif count > 1:
        raise ValueError(f"positions of {count} axes need axes")
    if not sound:
        there = check_tensors(("frequencies", frequencies, torch.float64, (pairs,)), ("axes", axes, _INT, (pairs,)),
                              ("positions", positions if tokens else None, _INT, None if positions is None else positions.shape))
        if there.index != device:
            raise ValueError(f"frequencies must be on the heads' device, got {there}")
    return at, stride, count, frequencies.data_ptr(), axis, pairs


def _weight(name: str, w, heads: int, dim: int, dtype, device: int) -> tuple[int, int]:
    """(address, stride of the heads) of a norm's weights."""
    if not isinstance(w, _Tensor) or w.shape not in ((dim,), (heads, dim)):
        raise ValueError(f"{name} must be a [{dim}] or [{heads}, {dim}] tensor")
    if w.dtype != dtype and w.dtype != torch.float32:
        raise ValueError(f"{name} must be {dtype} or float32, got {w.dtype}")
    if w.stride(-1) != 1 or w.get_device() != device:
        if check_tensors((name, w, w.dtype, w.shape)).index != device:
            raise ValueError(f"{name} must be on the heads' device, got {w.device}")
    return w.data_ptr(), w.stride(0) if w.ndim == 2 and heads > 1 else 0


def _weights(q_weight, q_heads: int, k_weight, kv_heads: int, dim: int, dtype, device: int) -> tuple[int, int, int, int, int]:
    """The fields (q weight, k weight, their strides, type)."""
    if q_weight is None and k_weight is None:
        return _NO_WEIGHTS
    q_at = q_stride = k_at = k_stride = 0
    if q_weight is not None:
        q_at, q_stride = _weight("q_weight", q_weight, q_heads, dim, dtype, device)
        kind = q_weight.dtype
    if k_weight is not None:
        k_at, k_stride = _weight("k_weight", k_weight, kv_heads, dim, dtype, device)
        if q_weight is not None and k_weight.dtype != kind:
            raise ValueError(f"k_weight must be {kind} as q_weight is, got {k_weight.dtype}")
        kind = k_weight.dtype
    return q_at, k_at, q_stride, k_stride, ekv_hip.dtype_code(kind)


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

    ``q_out`` and ``k_out`` may be ``query`` and ``key`` themselves; their heads overlap nothing else, nor each other.
    Types, head dims and limits as ``ekv_rotate_heads`` documents them.  ``stream``: the call launches and allocates as
    under ``torch.cuda.stream(stream)``; the caller orders it after the work that makes its inputs.  No gradient is
    taken through the call."""
    q_shape, dtype, device, q_at, q_token, q_head, sound = _look("query", query)
    tokens, q_heads, dim = q_shape
    k_shape, kv_heads, k_at, k_token, k_head = None, 0, 0, 0, 0
    if key is not None:
        k_shape, k_type, k_device, k_at, k_token, k_head, k_sound = _look("key", key)
        k_tokens, kv_heads, k_dim = k_shape
        if k_tokens != tokens or k_dim != dim:
            raise ValueError(f"key must be a [{tokens}, heads, {dim}] tensor, got {tuple(k_shape)}")
        sound = sound and k_sound and k_type is dtype and k_device == device
    elif k_out is not None or k_weight is not None:
        raise ValueError("k_out and k_weight need a key")
    if frequencies is not None and positions is None:
        raise ValueError("frequencies need positions")
    if not sound or device < 0 or dtype not in _HEAD_TYPES:
        if tokens == 0:  # no rows to be contiguous: an empty tensor's strides may be anything
            query, key = query.new_empty(q_shape), None if key is None else key.new_empty(k_shape)
        check_tensors(("query", query, _HEAD_TYPES, q_shape), ("key", key, dtype, k_shape), ("q_out", q_out, dtype, q_shape),
                      ("k_out", k_out, dtype, k_shape))
    at, stride, count, turning, axis, pairs = _turns(tokens, dim, positions, frequencies, axes, device)
    q_weighs, k_weighs, q_step, k_step, w_type = _NO_WEIGHTS if q_weight is None and k_weight is None else \
        _weights(q_weight, q_heads, k_weight, kv_heads, dim, dtype, device)
    context, handle = ekv_hip.beside(stream, query)
    with context or _HERE:
        # an output made here is contiguous
        if q_out is None:
            q_out = torch.empty(tokens, q_heads, dim, dtype=dtype, device=query.device)
            qo_at, qo_token, qo_head = q_out.data_ptr(), q_heads * dim, dim
        else:
            qo_at, qo_token, qo_head = _output("q_out", q_out, dtype, q_shape, query)
        ko_at = ko_token = ko_head = 0
        if key is not None:
            if k_out is None:
                k_out = torch.empty(tokens, kv_heads, dim, dtype=dtype, device=query.device)
                ko_at, ko_token, ko_head = k_out.data_ptr(), kv_heads * dim, dim
            else:
                ko_at, ko_token, ko_head = _output("k_out", k_out, dtype, k_shape, query)
        arguments = _pack(
            q_at, q_token, q_head, k_at, k_token, k_head, qo_at, qo_token, qo_head, ko_at, ko_token, ko_head, at,
            stride, turning, axis, q_weighs, k_weighs, q_step, k_step, ekv_hip.dtype_code(dtype), w_type, tokens, q_heads,
            kv_heads, dim, pairs, count, 1 if adjacent else 0, rotary_scale, eps, weight_offset)
        status = (ekv_hip._lib or ekv_hip.load()).ekv_rotate_heads(arguments, handle)
    if status:
        ekv_hip.check(status, "ekv_rotate_heads")
    return q_out, k_out
