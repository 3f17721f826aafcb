"""Tokens on their way into a paged cache, the norms of their heads with the rotation of their positions, and positions
of several axes: what is measured, and the plain form of each.

``append``  a batch's new keys and values go into its rows' pages, the keys rotated by their positions, and the queries
            beside them; an evicting cache's running scores and positions of the new slots are set in the same pass.
``norm``    root-mean-square norms of each query and key head and the rotation, without a cache.
``axes``    rotations whose pairs follow several axes (time, height, width), without a cache or on the way into one.

Sizes are this repository's: the 4-row fp32 check, the Llama-3-8B decode shape (32 query and 8 KV heads of 128,
16-token blocks, 512 to 8192 tokens), the fp8 step with its 32-token blocks; or generic ones.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}
ELEMENT = {"fp32": 4, "f16": 2, "bf16": 2, "fp8": 1}
FP8_SCALE = 6.0 / 448.0  # N(0, 1) fills the e4m3 range up to 6 sigma


def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


# -- cases ---------------------------------------------------------------------------------------------


def listed():
    heads = {"q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "adjacent": False, "base": 500000.0, "norm": "none",
             "axes": 1, "interleaved": False}
    append = {"op": "append", **heads, "block": 16, "dtype": "bf16", "kv": "bf16", "queries": 1, "singles": False,
              "pad": 0, "evicting": False}
    norm = {"op": "norm", **heads, "dtype": "bf16", "norm": "shared"}
    axes = {**heads, "axes": 3}
    return [
        # a few short requests in fp32, the correctness configuration: launches and host time are all of it
        dict(append, name="append_small_fp32", rows=4, low=17, high=512, q_heads=8, kv_heads=2, dim=64, rot=64,
             base=10000.0, dtype="fp32", kv="fp32"),
        # one interactive request with a long conversation: a decode step's latency
        dict(append, name="append_one_row", rows=1, low=8192, high=8192),
        # the ordinary decode step of a batch: a token a row, each into a page of its own
        dict(append, name="append_decode", rows=128, low=512, high=8192),
        # four drafted tokens a request of an evicting cache, whose slots are no positions; half the dimensions rotate,
        # in adjacent pairs, behind norms
        dict(append, name="append_drafts_f16", rows=200, low=64, high=1024, queries=4, dtype="f16", kv="f16", rot=64,
             adjacent=True, norm="shared", evicting=True),
        # prompt chunks among single tokens into an fp8 cache of 32-token blocks, the batch padded to a captured size
        dict(append, name="append_mixed_fp8", rows=64, low=2048, high=8192, queries=2048, singles=True, block=32,
             kv="fp8", pad=100),
        # whole prompts, the most bytes
        dict(append, name="append_prompts", rows=8, low=8192, high=8192, queries=8192),
        # the norms of a decode step, for a cache of another kind
        dict(norm, name="norm_decode", tokens=128),
        # a long prompt's norms
        dict(norm, name="norm_prompt", tokens=16384),
        # weights of each head, wide heads of which half rotate, an odd count of tokens
        dict(norm, name="norm_wide_f16", tokens=777, q_heads=16, kv_heads=4, dim=256, rot=128, adjacent=True,
             norm="heads", dtype="f16"),
        # the frames of a video through an encoder: every head a query's and a key's, 8 frames of 36 x 52 patches
        dict(axes, op="axes", name="axes_video_f16", cached=False, tokens=14976, q_heads=16, kv_heads=16, dim=80, rot=80,
             base=10000.0, dtype="f16", frame=36, width=52),
        # text and images on their way into the cache, seven query heads a KV head
        dict(axes, op="axes", name="axes_prompts", cached=True, rows=6, low=700, high=2500, queries=2500, singles=False,
             pad=0, evicting=False, q_heads=28, kv_heads=4, block=16, dtype="bf16", kv="bf16", base=1000000.0,
             frame=24, width=32),
        # and the tokens that answer, one a row, the axes taking turns over the pairs
        dict(axes, op="axes", name="axes_decode_fp8", cached=True, rows=64, low=512, high=4096, queries=1, singles=False,
             pad=0, evicting=False, q_heads=28, kv_heads=4, block=32, dtype="bf16", kv="fp8", base=1000000.0,
             norm="shared", interleaved=True, frame=24, width=32),
    ]


def _log(rng, low, high):
    """A whole number spread over the logarithm of low .. high."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "append", "append", "norm", "norm", "axes", "axes"])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    case = {"op": op, "kv_heads": kv_heads, "q_heads": kv_heads * rng.choice([1, 2, 3, 4, 7, 8]),
            "adjacent": rng.random() < 0.3, "base": rng.choice([10000.0, 500000.0]),
            "norm": rng.choice(["none", "none", "shared", "heads"]), "axes": 1, "interleaved": False,
            "dtype": rng.choice(["bf16", "bf16", "f16", "fp32"])}
    if op == "norm":
        case["norm"] = rng.choice(["shared", "shared", "heads"])
    if op == "axes":
        case.update(axes=rng.choice([2, 3, 3, 4]), interleaved=rng.random() < 0.4, cached=rng.random() < 0.5,
                    frame=_log(rng, 4, 48), width=_log(rng, 4, 64))
    if op == "append" or op == "axes" and case["cached"]:
        high = _log(rng, 16, 16384)
        case.update(dim=rng.choice([32, 64, 128, 128, 256]), rows=_log(rng, 1, 256), low=max(1, high // rng.choice([1, 4, 16])),
                    high=high, queries=min(high, rng.choice([1, 1, 2, 5, _log(rng, 6, 8192)])), singles=rng.random() < 0.3,
                    pad=rng.choice([0, 0, 1, 37]), evicting=op == "append" and rng.random() < 0.3,
                    block=rng.choice([8, 16, 16, 24, 32, 64]), kv=rng.choice([case["dtype"], case["dtype"], "fp8"]))
        if case["queries"] == 1:
            case["pad"] = 0
    else:
        case.update(dim=rng.choice([32, 64, 80, 96, 112, 128, 128, 192, 256]), tokens=_log(rng, 1, 32768))
    case["rot"] = rng.choice([case["dim"], case["dim"], max(16, case["dim"] // 32 * 16)])
    return _within(case)


def _within(case):
    """The case made smaller until it moves no more than the largest listed one and its plain form fits the card."""
    def over(c):
        moved = work(c)["bytes"]
        pool = c["rows"] * c["high"] * c["kv_heads"] * c["dim"] * 2 if "rows" in c else 0
        return moved > 8e8 or pool > 1.5e9

    while over(case):
        key = "tokens" if "tokens" in case else max(
            ("rows", "high", "queries"), key=lambda k: case[k] / {"rows": 4, "high": 1024, "queries": 256}[k])
        case[key] = max(1, case[key] * 2 // 3)
        if "rows" in case:
            case["low"] = min(case["low"], case["high"])
            case["queries"] = min(case["queries"], case["high"])
    return case


# -- the structure of a batch (whole numbers, from the seed alone) ----------------------------------------


def _structure(case, seed):
    """Lengths (the new tokens among them) and counts of new tokens: the sizes go by the case, which row has which by
    the seed, so that outputs have one shape whatever the seed."""
    fixed, rng = np.random.default_rng(17), np.random.default_rng((seed, 17))
    rows, t = case["rows"], case["queries"]
    lens = fixed.integers(case["low"], case["high"] + 1, size=rows)
    lens[0] = case["high"]
    if t > 8:  # prompt chunks are ragged; a row without new tokens among five or more
        counts = fixed.integers(max(1, t // 4), t + 1, size=rows)
        counts[0] = t
        if rows >= 5:
            counts[rows - 1] = 0
        if case["singles"]:  # most rows have a token
            counts = np.where(np.arange(rows) % 8 == 0, counts, 1)
    else:
        counts = np.full(rows, t)
    counts = np.minimum(counts, lens)
    order = rng.permutation(rows)
    return lens[order], counts[order]


def _sections(case):
    """The axis of each rotated pair: a quarter of them the first axis's and the rest shared evenly, as runs or in turn."""
    pairs, axes = case["rot"] // 2, case["axes"]
    if case["interleaved"]:
        return np.arange(pairs) % axes
    first = pairs // 4
    return np.concatenate([np.zeros(first, int), 1 + np.arange(pairs - first) * (axes - 1) // (pairs - first)])


def prepare(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    cached = "rows" in case
    q_heads, kv_heads, d, pairs = case["q_heads"], case["kv_heads"], case["dim"], case["rot"] // 2
    dtype = DTYPES[case["dtype"]]
    state = {"cached": cached, "adjacent": case["adjacent"], "eps": 1e-6, "axes": None, "positions": None}
    if cached:
        lens, counts = _structure(case, seed)
        starts = np.concatenate([[0], np.cumsum(counts)])
        tokens = int(starts[-1]) + case["pad"]
    else:
        tokens = case["tokens"]
    # what the projection leaves: queries, keys and values of a token beside each other, the values around a mean
    parts = q_heads + (2 if cached else 1) * kv_heads
    packed = torch.empty(tokens, parts, d, dtype=dtype, device=dev)
    mean = 0.5 * torch.randn(kv_heads, d, generator=gen, device=dev)
    step = max(1, (1 << 26) // (parts * d))
    for a in range(0, tokens, step):
        part = torch.randn(min(step, tokens - a), parts, d, generator=gen, device=dev)
        if cached:
            part[:, q_heads + kv_heads:] += mean
        packed[a:a + step] = part.to(dtype)
    state.update(query=packed[:, :q_heads], key=packed[:, q_heads:q_heads + kv_heads])
    # radians a position, as a model's configuration gives them
    state["frequencies"] = torch.from_numpy(float(case["base"]) ** -(np.arange(pairs) / pairs)).to(dev)
    state["q_weight"] = state["k_weight"] = None
    if case["norm"] != "none":
        for name, heads in (("q_weight", q_heads), ("k_weight", kv_heads)):
            shape = (heads, d) if case["norm"] == "heads" else (d,)
            state[name] = (1.0 + 0.2 * torch.randn(shape, generator=gen, device=dev)).to(dtype)
    if case["axes"] > 1:
        # patches of frames: time, then the place in a frame (a fourth axis counts them), somewhere in a conversation
        n = np.arange(tokens) + 7 * (seed % 100)
        tall, wide = case["frame"], case["width"]
        grid = np.stack([n // (tall * wide), n // wide % tall, n % wide, n])[:case["axes"]]
        state["positions"] = torch.from_numpy(grid.astype(np.int32) + 1000).to(dev)
        state["axes"] = torch.from_numpy(_sections(case).astype(np.int32)).to(dev)
    elif not cached:
        state["positions"] = torch.arange(tokens, dtype=torch.int32, device=dev) + 100000 + seed % 1000
    if not cached:
        return state

    bs = case["block"]
    fp8 = case["kv"] == "fp8"
    need = (lens + bs - 1) // bs
    width = -(-case["high"] // bs)
    pool = int(need.sum()) + 1  # page 0 is nobody's
    ids = torch.randperm(pool - 1, generator=gen, device=dev).to(torch.int32) + 1
    have = torch.from_numpy(need).to(dev)
    at, j = torch.cumsum(have, 0) - have, torch.arange(width, device=dev)
    live = j[None] < have[:, None]
    table = torch.where(live, ids[torch.where(live, at[:, None] + j[None], 0)], 0).to(torch.int32).contiguous()
    cache = torch.empty(pool, 2, bs, kv_heads, d, dtype=DTYPES[case["kv"]], device=dev)
    step = max(1, (1 << 27) // (2 * bs * kv_heads * d))
    for a in range(0, pool, step):
        part = torch.randn(min(step, pool - a), 2, bs, kv_heads, d, generator=gen, device=dev)
        if fp8:
            part = (part / FP8_SCALE).clamp_(-448.0, 448.0)
        cache[a:a + step] = part.to(cache.dtype)
    state.update(value=packed[:, q_heads + kv_heads:], cache=cache, table=table,
                 lens=torch.from_numpy(lens.astype(np.int32)).to(dev), max_query=max(1, int(counts.max())),
                 q_start=None if case["queries"] == 1 and not case["pad"] else torch.from_numpy(starts.astype(np.int32)).to(dev),
                 k_scale=FP8_SCALE if fp8 else 1.0, v_scale=FP8_SCALE if fp8 else 1.0, seen=None, scores=None,
                 slot_positions=None, all_scores=None, all_positions=None)
    if case["evicting"]:
        # a cache that let tokens go: the next position is past the next slot; running scores of what it holds
        rng = np.random.default_rng((seed, 19))
        gone = torch.from_numpy(rng.integers(0, 200000, size=case["rows"])).to(dev)
        state["seen"] = (state["lens"] + gone).to(torch.int32)
        shape = (case["rows"] + 1, kv_heads, width * bs)  # a row more than there are, for tokens of no row
        state["all_scores"] = torch.exp(2.0 * torch.randn(shape, generator=gen, device=dev) - 3.0)
        state["all_positions"] = torch.randint(0, 200000, shape, generator=gen, device=dev, dtype=torch.int32)
        state.update(scores=state["all_scores"][:-1], slot_positions=state["all_positions"][:-1])
    return state


# -- one pass ---------------------------------------------------------------------------------------------


def run(state):
    if state["cached"]:
        return _append_own(state) if own else _append_plain(state)
    return _rotate_own(state) if own else _rotate_plain(state)


def _package():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sigmod-kvscope_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)


def _rotate_own(s):
    _package()
    from runtime.rotary import rotate_heads

    query, key = rotate_heads(s["query"], s["key"], s["positions"], s["frequencies"], axes=s["axes"],
                              adjacent=s["adjacent"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=s["eps"])
    return {"query": query, "key": key}


def _append_own(s):
    _package()
    from runtime.append import append_tokens

    query = append_tokens(s["cache"], s["table"], s["lens"], s["key"], s["value"], q_start=s["q_start"],
                          max_query=s["max_query"], query=s["query"], positions=s["positions"],
                          frequencies=s["frequencies"], axes=s["axes"], adjacent=s["adjacent"], q_weight=s["q_weight"],
                          k_weight=s["k_weight"], eps=s["eps"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                          seen=s["seen"], scores=s["scores"], slot_positions=s["slot_positions"])
    return _answer(s, query)


def _answer(s, query):
    answer = {"query": query, "cache": s["cache"]}
    if s["scores"] is not None:
        answer.update(scores=s["scores"], slot_positions=s["slot_positions"])
    return answer


# -- the plain forms: in float32, angles in float64 --------------------------------------------------------


def _turned(s, positions):
    """Cosines and sines ``[tokens, 1, pairs]`` of positions ``[axes, tokens]``."""
    at = positions.double()
    at = at[0][:, None] if s["axes"] is None else at[s["axes"].long()].t()
    angle = at * s["frequencies"][None]
    return torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]


def _heads(s, x, weight, cos, sin):
    """Heads ``[tokens, heads, dim]`` normed (with a weight) and rotated, in float32."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + s["eps"]) * weight.float()
    pairs = cos.shape[-1]
    turning, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if s["adjacent"]:
        a, b = turning[..., 0::2], turning[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = turning[..., :pairs], turning[..., pairs:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _rotate_plain(s):
    positions = s["positions"] if s["positions"].ndim == 2 else s["positions"][None]
    cos, sin = _turned(s, positions)
    return {"query": _heads(s, s["query"], s["q_weight"], cos, sin).to(s["query"].dtype),
            "key": _heads(s, s["key"], s["k_weight"], cos, sin).to(s["key"].dtype)}


def _append_plain(s):
    cache, table, lens = s["cache"], s["table"].long(), s["lens"].long()
    dev, rows, tokens, bs = cache.device, table.shape[0], s["key"].shape[0], cache.shape[2]
    start = torch.arange(rows + 1, device=dev) if s["q_start"] is None else s["q_start"].long()
    count = start[1:] - start[:-1]
    token = torch.arange(tokens, device=dev)
    row = (torch.searchsorted(start, token, right=True) - 1).clamp(0, rows - 1)
    nth = token - start[row]
    live = (nth >= 0) & (nth < count[row])
    slot = torch.where(live, lens[row] - count[row] + nth, 0)
    index = slot if s["seen"] is None else torch.where(live, s["seen"].long()[row] - count[row] + nth, 0)
    cos, sin = _turned(s, index[None] if s["positions"] is None else s["positions"])
    query = _heads(s, s["query"], s["q_weight"], cos, sin)
    query = torch.where(live[:, None, None], query, 0.0).to(s["query"].dtype)
    key = _heads(s, s["key"], s["k_weight"], cos, sin) / s["k_scale"]
    value = s["value"].float() / s["v_scale"]
    raw = cache
    if cache.dtype == torch.float8_e4m3fn:
        key, value, raw = key.clamp(-448.0, 448.0), value.clamp(-448.0, 448.0), cache.view(torch.uint8)
    page = torch.where(live, table[row, slot // bs], 0)
    off = torch.where(live, slot % bs, 0)
    for part, new in ((0, key), (1, value)):
        new = new.to(cache.dtype)
        new = new.view(torch.uint8) if raw is not cache else new
        # a token of no row writes page 0's first slot with itself
        raw[page, part, off] = torch.where(live[:, None, None], new, raw[0, part, 0])
    if s["scores"] is not None:
        into = torch.where(live, row, rows)
        s["all_scores"][into, :, slot] = 0.0
        s["all_positions"][into, :, slot] = index.int()[:, None]
    return _answer(s, query)


# -- what a pass cannot do without ------------------------------------------------------------------------


def work(case):
    """Expected over the seeds: lengths and counts are uniform between their bounds."""
    e, d, q_heads, kv_heads = ELEMENT[case["dtype"]], case["dim"], case["q_heads"], case["kv_heads"]
    if "rows" in case:
        t = case["queries"] if case["queries"] <= 8 else 0.625 * case["queries"]
        if case["singles"] and case["queries"] > 8:
            t = (t + 7) / 8
        tokens = case["rows"] * min(t, (case["low"] + case["high"]) / 2)
        moved = tokens * d * (q_heads * 2 * e + 2 * kv_heads * (e + ELEMENT[case["kv"]])) + case["pad"] * d * q_heads * e
        moved += tokens * 4 * case["axes"] * (case["axes"] > 1) + case["rows"] * 12
        if case["evicting"]:
            moved += tokens * kv_heads * 8
    else:
        tokens = case["tokens"]
        moved = tokens * (d * (q_heads + kv_heads) * 2 * e + 4 * case["axes"])
    moved += case["rot"] // 2 * 8
    heads = tokens * (q_heads + kv_heads)
    return {"bytes": moved, "flops": heads * (3.0 * case["rot"] + (4.0 * d if case["norm"] != "none" else 0.0))}


# -- the definitions in 64 bits ---------------------------------------------------------------------------


def _spun(x, weight, eps, angle, adjacent):
    """Heads ``[n, heads, dim]`` in float64: over their root mean square, times the weight, and each pair of them a complex
    number turned by its angle ``[n, pairs]``."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    pairs = angle.shape[1]
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    if adjacent:
        z = torch.view_as_real(torch.view_as_complex(x[..., :2 * pairs].unflatten(-1, (pairs, 2)).contiguous()) * turn)
        front = z.reshape(*x.shape[:2], 2 * pairs)
    else:
        z = torch.complex(x[..., :pairs].contiguous(), x[..., pairs:2 * pairs].contiguous()) * turn
        front = torch.cat([z.real, z.imag], -1)
    return torch.cat([front, x[..., 2 * pairs:]], -1)


def _angles(s, positions):
    """Angles ``[n, pairs]`` of positions ``[axes, n]``, pair by pair."""
    f = s["frequencies"].tolist()
    axis = [0] * len(f) if s["axes"] is None else s["axes"].tolist()
    return torch.stack([positions[a].double() * w for a, w in zip(axis, f)], 1)


def exact(case, seed):
    s = prepare(case, seed)
    if not s["cached"]:
        angle = _angles(s, s["positions"].reshape(-1, s["key"].shape[0]))
        return {"query": _spun(s["query"], s["q_weight"], s["eps"], angle, s["adjacent"]),
                "key": _spun(s["key"], s["k_weight"], s["eps"], angle, s["adjacent"])}
    cache, table, bs = s["cache"].double(), s["table"], s["cache"].shape[2]
    rows, dev = table.shape[0], cache.device
    query = torch.zeros(s["query"].shape, dtype=torch.float64, device=dev)
    scores = None if s["scores"] is None else s["scores"].double()
    start = list(range(rows + 1)) if s["q_start"] is None else s["q_start"].tolist()
    lens = s["lens"].tolist()
    seen = lens if s["seen"] is None else s["seen"].tolist()
    for r in range(rows):
        a, b = start[r], start[r + 1]
        if a == b:
            continue
        new = torch.arange(lens[r] - (b - a), lens[r], device=dev)
        where = new + (seen[r] - lens[r]) if s["positions"] is None else s["positions"][:, a:b]
        angle = _angles(s, where.reshape(-1, b - a))
        query[a:b] = _spun(s["query"][a:b], s["q_weight"], s["eps"], angle, s["adjacent"])
        key = _spun(s["key"][a:b], s["k_weight"], s["eps"], angle, s["adjacent"]) / s["k_scale"]
        value = s["value"][a:b].double() / s["v_scale"]
        page = table[r].long()[new // bs]
        cache[page, 0, new % bs], cache[page, 1, new % bs] = key, value
        if scores is not None:
            scores[r, :, lens[r] - (b - a):lens[r]] = 0.0
    answer = {"query": query, "cache": cache}
    if scores is not None:
        answer.update(scores=scores, slot_positions=None)
    return answer
