"""Attention over a paged cache whose rows share prefixes, the weight each cached token accumulates, and
the eviction of the tokens that accumulated least: what is measured, and the plain form of each.

``attend``   one layer's attention of a batch: every row reads its group's shared prefix and its own pages.
``observe``  the same call adding each own token's attention weight to its running score.
``evict``    a budget of tokens a row: the heaviest, the first and the newest stay; survivors from behind
             the budget move into the freed slots.

Sizes are this repository's: the 4-row fp32 check, the Llama-3-8B decode shape (32 query and 8 KV heads of
128, 16-token blocks, 512 to 8192 tokens), the fp8 step with its 32-token blocks; or generic ones.
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
NEG = float("-inf")


def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


# -- cases ---------------------------------------------------------------------------------------------


def listed():
    attend = {"op": "attend", "kv_heads": 8, "group": 4, "dim": 128, "block": 16, "dtype": "bf16", "queries": 1,
              "groups": 0, "prefix": 0, "empty": False}
    evict = {"op": "evict", "kv_heads": 8, "dim": 128, "block": 16, "dtype": "bf16", "sinks": 4, "recent": 32}
    return [
        # a few short requests in fp32, the correctness configuration: launches and host time are all of it
        dict(attend, name="attend_small_fp32", rows=4, low=17, high=512, kv_heads=2, dim=64, dtype="fp32"),
        # one interactive request with a long conversation: the decode step's latency, nothing to batch
        dict(attend, name="attend_one_row", rows=1, low=8192, high=8192),
        # the ordinary decode step of a batch with nothing shared: all bandwidth
        dict(attend, name="attend_decode", rows=128, low=512, high=8192),
        # a service whose requests share one long system prompt and have short turns of their own
        dict(attend, name="attend_prefix", rows=128, low=16, high=1024, groups=1, prefix=8192),
        # two document prompts asked by many, four drafted tokens a request: the most arithmetic
        dict(attend, name="attend_prefix_drafts_f16", rows=200, low=5, high=600, queries=4, groups=2, prefix=32768,
             dtype="f16"),
        # ragged prompt chunks behind a shared instruction prefix
        dict(attend, name="attend_chunk", rows=5, low=700, high=3000, queries=1024, groups=1, prefix=1999),
        # an fp8 cache in 32-token blocks, a shared prefix, one request still without tokens of its own
        dict(attend, name="attend_fp8", rows=64, low=512, high=8192, block=32, groups=3, prefix=2048, dtype="fp8",
             empty=True),
        # decode with the running scores kept, as an evicting cache runs every step
        dict(attend, name="observe_decode", op="observe", rows=128, low=512, high=4128, groups=1, prefix=512),
        # the scores' start: prompt chunks of a model with 7 query heads a KV head of 64
        dict(attend, name="observe_chunk_f16", op="observe", rows=3, low=300, high=2047, queries=777, kv_heads=4,
             group=7, dim=64, dtype="f16"),
        # eviction of a small batch
        dict(evict, name="evict_small_fp32", rows=4, low=17, high=512, budget=128, kv_heads=2, dim=64, dtype="fp32"),
        # the steady state: a few tokens past the budget every few steps
        dict(evict, name="evict_step", rows=128, low=4097, high=4128, budget=4096),
        # a budget cut in the middle of the run: half of the long requests' tokens go
        dict(evict, name="evict_cut", rows=128, low=512, high=8192, budget=2048),
    ]


def _log(rng, low, high):
    """A whole number spread over the logarithm of low .. high."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "observe", "observe", "evict", "evict"])
    case = {"op": op, "rows": _log(rng, 1, 256), "kv_heads": rng.choice([1, 2, 4, 8]),
            "dim": rng.choice([32, 64, 128, 128, 256]), "block": rng.choice([8, 16, 16, 24, 32, 64]),
            "dtype": rng.choice(["bf16", "bf16", "f16", "fp8", "fp32"])}
    high = _log(rng, 16, 16384)
    low = max(1, high // rng.choice([1, 4, 16]))
    if op == "evict":
        case.update(low=low, high=high, budget=max(1, int(high * rng.uniform(0.1, 1.0))),
                    sinks=rng.choice([0, 1, 4]), recent=rng.choice([0, 16, 64]))
    else:
        case.update(low=low, high=high, group=rng.choice([1, 2, 3, 4, 7, 8, 16]),
                    queries=rng.choice([1, 1, 1, 2, 5, _log(rng, 6, 1024)]), groups=0, prefix=0,
                    empty=rng.random() < 0.25)
        if rng.random() < 0.6:
            case.update(groups=min(case["rows"], rng.choice([1, 1, 2, 5])), prefix=_log(rng, 16, 32768))
    return _within(case)


def _within(case):
    """The case made smaller until it costs no more than the largest listed one (a quarter of its
    arithmetic in fp32) and its dense plain form about 8 GB."""
    def over(c):
        w = work(c)
        if w["bytes"] > 2.2e9 or w["flops"] > (1.2e11 if c["dtype"] == "fp32" else 4e11):
            return True
        heads = c["kv_heads"]
        dense = c["rows"] * c["high"] * heads * c["dim"] * 4
        if c["op"] != "evict":
            m = c["rows"] * c["queries"] * c["group"] * heads
            dense = max(dense, m * c["high"] * 4, m * c["prefix"] * 4)
        return dense > 8e9

    while over(case):
        key = max(("rows", "high", "prefix", "queries"), key=lambda k: case.get(k, 0) / {"rows": 8, "high": 512,
                  "prefix": 512, "queries": 64}[k])
        case[key] = max(1, case[key] * 2 // 3)
        case["low"] = min(case["low"], case["high"])
        if "groups" in case:
            case["groups"] = min(case["groups"], case["rows"])
        if "budget" in case:
            case["budget"] = max(1, min(case["budget"], case["high"]))
    return case


# -- the structure of a batch (whole numbers, from the seed alone) ----------------------------------------


def _structure(case, seed):
    """Lengths, query counts and group borders of the batch, as numpy arrays: the sizes go by the case, which
    row has which by the seed, so that outputs have one shape whatever the seed."""
    fixed, rng = np.random.default_rng(11), np.random.default_rng((seed, 11))
    rows = case["rows"]
    lens = fixed.integers(case["low"], case["high"] + 1, size=rows)
    lens[0] = case["high"]
    order = rng.permutation(rows)
    if case["op"] == "evict":
        return {"lens": lens[order]}
    if case["empty"]:
        lens[rows - 1] = 0
    t = case["queries"]
    if t > 8:  # prompt chunks are ragged
        counts = fixed.integers(max(1, t // 4), t + 1, size=rows)
        counts[0] = t
    else:
        counts = np.full(rows, t)
    counts = np.where(lens > 0, np.minimum(counts, lens), 1)  # the queries are among the row's own tokens
    s = {"lens": lens[order], "counts": counts[order]}
    if case["groups"]:
        g = case["groups"]
        cuts = np.sort(rng.choice(np.arange(1, rows), size=g - 1, replace=False)) if g > 1 else np.zeros(0, int)
        s["borders"] = np.concatenate([[0], cuts, [rows]]).astype(np.int64)
        s["prefix_lens"] = fixed.integers(max(1, case["prefix"] * 3 // 4), case["prefix"] + 1, size=g)
        s["prefix_lens"][0] = case["prefix"]
        s["prefix_lens"] = s["prefix_lens"][rng.permutation(g)]
    return s


def _pages(lens, block):
    return (np.asarray(lens, np.int64) + block - 1) // block


def prepare(case, seed):
    dev, bs = _device(), case["block"]
    s = _structure(case, seed)
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    rows, heads, d = case["rows"], case["kv_heads"], case["dim"]
    dtype = DTYPES[case["dtype"]]
    width = int(_pages([case["high"]], bs)[0])
    need = _pages(s["lens"], bs)
    prefix = s.get("prefix_lens")
    pneed = _pages(prefix, bs) if prefix is not None else np.zeros(0, np.int64)
    pool = int(need.sum() + pneed.sum()) + 1  # page 0 is nobody's
    ids = torch.randperm(pool - 1, generator=gen, device=dev).to(torch.int32) + 1

    def tables(counts, w, first):
        c = torch.from_numpy(counts).to(dev)
        at = torch.cumsum(c, 0) - c + first
        j = torch.arange(w, device=dev)
        live = j[None] < c[:, None]
        where = torch.where(live, at[:, None] + j[None], 0)
        return torch.where(live, ids[where], 0).to(torch.int32).contiguous()

    # keys and values N(0, 1), the values around a mean of their head and channel, as projections with a bias give
    cache = torch.empty(pool, 2, bs, heads, d, dtype=dtype, device=dev)
    mean = 0.5 * torch.randn(heads, d, generator=gen, device=dev)
    step = max(1, (1 << 27) // (2 * bs * heads * d))
    fp8 = case["dtype"] == "fp8"
    for a in range(0, pool, step):
        part = torch.randn(min(step, pool - a), 2, bs, heads, d, generator=gen, device=dev)
        part[:, 1] += mean
        if fp8:
            part = (part / FP8_SCALE).clamp_(-448.0, 448.0)
        cache[a:a + step] = part.to(dtype)
    state = {"op": case["op"], "cache": cache, "table": tables(need, width, 0), "high": case["high"], "block": bs,
             "lens": torch.from_numpy(s["lens"].astype(np.int32)).to(dev)}
    capacity = width * bs
    live = torch.arange(capacity, device=dev)[None] < state["lens"][:, None]
    if case["op"] == "evict":
        # scores as attention leaves them: a few tokens hold most of the weight, many hold next to none
        raw = torch.exp(3.0 * torch.randn(rows, heads, capacity, generator=gen, device=dev) - 4.0)
        raw = torch.where(raw < 1e-4, 0.0, raw)
        state["scores"] = torch.where(live[:, None], raw, 0.0)
        # the positions that the slots hold after earlier evictions: distinct, the newest ones at the end
        jitter = torch.randint(0, 3, (rows, heads, capacity), generator=gen, device=dev)
        pos = torch.arange(capacity, device=dev) * 3 + jitter
        state["positions"] = torch.where(live[:, None], pos, -1).to(torch.int32)
        state["seen"] = state["lens"] * 3
        state["budget"] = torch.full((rows,), case["budget"], dtype=torch.int32, device=dev)
        state.update(sinks=case["sinks"], recent=case["recent"] * 3)
        return state
    starts = np.concatenate([[0], np.cumsum(s["counts"])])
    qtype = torch.bfloat16 if fp8 else dtype
    # queries of sigma 1.5: logits spread enough that some keys stand out
    query = 1.5 * torch.randn(int(starts[-1]), heads * case["group"], d, generator=gen, device=dev)
    state.update(query=query.to(qtype), scale=d ** -0.5, max_query=int(s["counts"].max()),
                 q_start=None if case["queries"] == 1 else torch.from_numpy(starts.astype(np.int32)).to(dev),
                 k_scale=FP8_SCALE if fp8 else 1.0, v_scale=FP8_SCALE if fp8 else 1.0, prefix_table=None,
                 prefix_lens=None, prefix_rows=None, longest_prefix=0, largest_group=0, scores=None, decay=1.0)
    if prefix is not None:
        state.update(prefix_table=tables(pneed, int(pneed.max()), int(need.sum())),
                     prefix_lens=torch.from_numpy(prefix.astype(np.int32)).to(dev),
                     prefix_rows=torch.from_numpy(s["borders"].astype(np.int32)).to(dev),
                     longest_prefix=int(prefix.max()), largest_group=int(np.diff(s["borders"]).max()))
    if case["op"] == "observe":
        old = torch.exp(2.0 * torch.randn(rows, heads, capacity, generator=gen, device=dev) - 3.0)
        state.update(scores=torch.where(live[:, None], old, 0.0), decay=0.98)
    return state


# -- one pass ---------------------------------------------------------------------------------------------


def run(state):
    if state["op"] == "evict":
        return _evict_own(state) if own else _evict_plain(state)
    return _attend_own(state) if own else _attend_plain(state)


def _package():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sigmod-kvscope_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)


def _attend_own(s):
    _package()
    from runtime.prefix_attention import prefix_attention

    out, lse = prefix_attention(
        s["query"], s["cache"], s["table"], s["lens"], s["scale"], q_start=s["q_start"], max_query=s["max_query"],
        prefix_table=s["prefix_table"], prefix_lens=s["prefix_lens"], prefix_rows=s["prefix_rows"],
        k_scale=s["k_scale"], v_scale=s["v_scale"], scores=s["scores"], decay=s["decay"])
    return {"out": out, "lse": lse} if s["scores"] is None else {"out": out, "lse": lse, "scores": s["scores"]}


def _evict_own(s):
    _package()
    from runtime.eviction import evict_tokens

    lens, scores, positions = evict_tokens(s["cache"], s["table"], s["lens"], s["scores"], s["positions"], s["budget"],
                                           s["seen"], recent=s["recent"], sinks=s["sinks"])
    return {"lens": lens, "scores": scores, "positions": positions, "cache": s["cache"]}


# -- the plain forms: dense, masked, in float32 -----------------------------------------------------------


def _dense(cache, table, length):
    """Keys and values ``[rows, kv_heads, length, dim]`` of the first ``length`` slots of each table row."""
    j = torch.arange(length, device=cache.device)
    page = table.long()[:, j // cache.shape[2]]
    both = cache[page, :, j % cache.shape[2]].float()  # [rows, length, 2, kv_heads, dim]
    return both[:, :, 0].transpose(1, 2).contiguous(), both[:, :, 1].transpose(1, 2).contiguous()


def _part(query, keys, values, visible, scale):
    """Maximum, sum and weighted values of one set of keys: query ``[b, h, m, d]``, visible ``[b, 1, m, n]``."""
    logits = torch.matmul(query, keys.transpose(2, 3).contiguous()) * scale
    logits = logits.masked_fill_(~visible, NEG)
    top = logits.amax(dim=3)
    weight = torch.exp(logits - torch.where(top == NEG, 0.0, top)[..., None])
    return top, weight.sum(dim=3), torch.matmul(weight, values), logits


def _attend_plain(s):
    cache, table, lens, query = s["cache"], s["table"], s["lens"].long(), s["query"]
    dev, (rows, heads, d) = cache.device, (table.shape[0], cache.shape[3], cache.shape[4])
    tokens, q_heads = query.shape[0], query.shape[1]
    group, longest = q_heads // heads, s["max_query"]
    start = torch.arange(rows + 1, device=dev) if s["q_start"] is None else s["q_start"].long()
    count = start[1:] - start[:-1]
    i = torch.arange(longest, device=dev)
    has = i[None] < count[:, None]  # [rows, longest]
    at = torch.where(has, start[:-1, None] + i[None], 0)
    scale = s["scale"] * s["k_scale"]

    # own pages: query i of a row with t queries sees slots up to len - t + i
    dense_q = query[at].float().reshape(rows, longest, heads, group, d)
    dense_q = dense_q.permute(0, 2, 1, 3, 4).reshape(rows, heads, longest * group, d)
    keys, values = _dense(cache, table, s["high"])
    j = torch.arange(s["high"], device=dev)
    valid = j[None] < lens[:, None]
    values = values * valid[:, None, :, None]
    sees = has[:, :, None] & valid[:, None] & (j[None, None] <= (lens - count)[:, None, None] + i[None, :, None])
    sees = sees[:, :, None].expand(rows, longest, group, s["high"]).reshape(rows, 1, longest * group, s["high"])
    top, total, mixed, logits = _part(dense_q, keys, values, sees, scale)

    if s["prefix_table"] is not None:
        # the prefixes: the rows of each group beside each other, padded to the largest group
        border, most = s["prefix_rows"].long(), s["largest_group"]
        groups = border.shape[0] - 1
        k = torch.arange(most, device=dev)
        member = border[:-1, None] + k[None]
        there = member < border[1:, None]
        gq = dense_q[torch.where(there, member, 0)]  # [groups, most, heads, m, d]
        m = longest * group
        gq = gq.transpose(1, 2).reshape(groups, heads, most * m, d)
        pkeys, pvalues = _dense(cache, s["prefix_table"], s["longest_prefix"])
        in_prefix = torch.arange(s["longest_prefix"], device=dev)[None] < s["prefix_lens"].long()[:, None]
        pvalues = pvalues * in_prefix[:, None, :, None]
        ptop, ptotal, pmixed, _ = _part(gq, pkeys, pvalues, in_prefix[:, None, None], scale)
        row = torch.arange(rows, device=dev)
        of = torch.searchsorted(border, row, right=True) - 1
        place = row - border[of]
        ptop = ptop.reshape(groups, heads, most, m)[of, :, place]
        ptotal = ptotal.reshape(groups, heads, most, m)[of, :, place]
        pmixed = pmixed.reshape(groups, heads, most, m, d)[of, :, place]
        both = torch.maximum(top, ptop)
        safe = torch.where(both == NEG, 0.0, both)
        a, b = torch.exp(top - safe), torch.exp(ptop - safe)
        top, total, mixed = both, a * total + b * ptotal, a[..., None] * mixed + b[..., None] * pmixed
    lse = top + torch.log(total)
    lse = torch.where(total > 0, lse, NEG)
    result = torch.where((total > 0)[..., None], mixed / total[..., None], 0.0) * s["v_scale"]

    # back to the tokens' order: token k is query k - start[row] of its row
    token = torch.arange(tokens, device=dev)
    row_of = torch.searchsorted(start, token, right=True) - 1
    nth = token - start[row_of]
    result = result.reshape(rows, heads, longest, group, d)[row_of, :, nth].reshape(tokens, q_heads, d)
    lse_out = lse.reshape(rows, heads, longest, group)[row_of, :, nth].reshape(tokens, q_heads)
    answer = {"out": result.to(query.dtype), "lse": lse_out.contiguous()}
    if s["scores"] is not None:
        weight = torch.exp(logits - torch.where(lse == NEG, 0.0, lse)[..., None]).sum(dim=2)
        scores = s["scores"][:, :, : s["high"]]
        scores.copy_(torch.where(valid[:, None], s["decay"] * scores + weight, scores))
        answer["scores"] = s["scores"]
    return answer


def _evict_plain(s):
    cache, table, lens, scores, positions = s["cache"], s["table"].long(), s["lens"].long(), s["scores"], s["positions"]
    dev, (rows, heads, capacity), bs = cache.device, scores.shape, cache.shape[2]
    slot = torch.arange(capacity, device=dev)
    live = (slot[None] < lens[:, None])[:, None].expand_as(scores)
    new = torch.minimum(lens, s["budget"].long().clamp_min(0))
    safe = (positions < s["sinks"]) | (positions >= (s["seen"].long() - s["recent"])[:, None, None])
    rank = torch.where(live, 1 + safe.long(), 0)
    # stable sorts, the lesser key first: by score, then by class
    order = torch.sort(torch.where(torch.isnan(scores), NEG, scores), dim=2, descending=True, stable=True).indices
    again = torch.sort(rank.gather(2, order), dim=2, descending=True, stable=True).indices
    order = order.gather(2, again)
    kept = torch.zeros(scores.shape, dtype=torch.bool, device=dev)
    kept.scatter_(2, order, (slot < new[:, None, None]).expand_as(kept))
    front = slot < new[:, None, None]
    hole, survivor = front & ~kept, ~front & kept
    nth_hole = torch.cumsum(hole, 2) - 1
    nth_survivor = torch.cumsum(survivor, 2) - 1
    listed_at = torch.zeros(rows, heads, capacity + 1, dtype=torch.long, device=dev)
    listed_at.scatter_(2, torch.where(survivor, nth_survivor, capacity), slot.expand_as(kept))
    source = torch.where(hole, listed_at.gather(2, nth_hole.clamp_min(0)), slot)
    new_scores = torch.where(front, scores.gather(2, source), 0.0)
    new_positions = torch.where(front, positions.gather(2, source), -1)
    # every front slot takes its source's key and value; what stays, and page 0, is written with itself
    front_t, source_t = front.transpose(1, 2), torch.where(front, source, 0).transpose(1, 2)  # [rows, capacity, 1 / heads]
    front_t = front_t.expand(rows, capacity, heads)
    r = torch.arange(rows, device=dev)[:, None, None]
    h = torch.arange(heads, device=dev)[None, None]
    to_page = torch.where(front_t, table[:, slot // bs][:, :, None], 0)
    to_off = torch.where(front_t, (slot % bs)[None, :, None], 0)
    from_page = torch.where(front_t, table[r, source_t // bs], 0)
    from_off = torch.where(front_t, source_t % bs, 0)
    raw = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache
    raw[to_page, :, to_off, h] = raw[from_page, :, from_off, h]
    return {"lens": new.to(torch.int32), "scores": new_scores, "positions": new_positions.to(torch.int32),
            "cache": cache}


# -- what a pass cannot do without ------------------------------------------------------------------------


def work(case):
    """Expected over the seeds: lengths are uniform between their bounds."""
    e, heads, d, rows = ELEMENT[case["dtype"]], case["kv_heads"], case["dim"], case["rows"]
    mean = (case["low"] + case["high"]) / 2
    if case["op"] == "evict":
        # a length n past the budget b moves the survivors behind b: about b (n - b) / n of them
        n = np.linspace(case["low"], case["high"], 257)
        moved = float(np.mean(np.where(n > case["budget"], case["budget"] * (n - case["budget"]) / n, 0.0)))
        capacity = math.ceil(case["high"] / case["block"]) * case["block"]
        return {"bytes": rows * heads * (mean * 8 + capacity * 8 + moved * 4 * d * e) + rows * capacity / case["block"] * 4,
                "flops": rows * heads * mean}
    q_heads, qe = heads * case["group"], 2 if case["dtype"] == "fp8" else e
    t = case["queries"] if case["queries"] <= 8 else 0.625 * case["queries"]
    t = min(t, mean)
    prefix = case["prefix"] * 0.94 if case["groups"] > 1 else case["prefix"] if case["groups"] else 0
    pairs = rows * t * (mean - t / 2 + prefix)
    moved = (rows * mean + case["groups"] * prefix) * heads * d * 2 * e
    moved += rows * t * q_heads * (d * 2 * qe + 4) + rows * mean / case["block"] * 4
    flops = 4.0 * d * q_heads * pairs
    if case["op"] == "observe":
        moved += rows * mean * heads * 8
    return {"bytes": moved, "flops": flops}


# -- the definitions in 64 bits ---------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return _evict_exact(state) if case["op"] == "evict" else _attend_exact(state)


def _tokens_of(cache, pages, n):
    """The first ``n`` tokens behind ``pages``: keys, values ``[kv_heads, n, dim]`` in float64."""
    bs = cache.shape[2]
    used = cache[pages[: -(-n // bs)].long()].double()  # [pages, 2, bs, heads, dim]
    flat = used.permute(1, 3, 0, 2, 4).reshape(2, cache.shape[3], -1, cache.shape[4])
    return flat[0, :, :n].contiguous(), flat[1, :, :n].contiguous()


def _attend_exact(s):
    cache, table, query = s["cache"], s["table"], s["query"]
    rows, heads = table.shape[0], cache.shape[3]
    group, d = query.shape[1] // heads, query.shape[2]
    start = list(range(rows + 1)) if s["q_start"] is None else s["q_start"].tolist()
    lens = s["lens"].tolist()
    out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
    lse = torch.full(query.shape[:2], NEG, dtype=torch.float64, device=query.device)
    scores = None if s["scores"] is None else s["scores"].double()
    borders = [] if s["prefix_rows"] is None else s["prefix_rows"].tolist()
    shared, current = None, -1
    for r in range(rows):
        n, t = lens[r], start[r + 1] - start[r]
        keys, values = _tokens_of(cache, table[r], n)
        p = 0
        for g in range(len(borders) - 1):
            if borders[g] <= r < borders[g + 1]:
                if g != current:
                    shared, current = _tokens_of(cache, s["prefix_table"][g], int(s["prefix_lens"][g])), g
                p = shared[0].shape[1]
                keys, values = torch.cat([shared[0], keys], 1), torch.cat([shared[1], values], 1)
        if p + n == 0 or t == 0:
            continue
        for a in range(0, t, 128):  # a slice of the queries at a time: few gigabytes of weights
            b = min(t, a + 128)
            q = query[start[r] + a:start[r] + b].double().reshape(b - a, heads, group, d)
            q = q.permute(1, 0, 2, 3).reshape(heads, (b - a) * group, d)
            x = torch.matmul(q, keys.transpose(1, 2).contiguous()).reshape(heads, b - a, group, p + n)
            x = x * (float(s["scale"]) * float(s["k_scale"]))
            last = torch.arange(a, b, device=x.device) + (n - t) + p
            x.masked_fill_((torch.arange(p + n, device=x.device)[None] > last[:, None])[None, :, None], NEG)
            z = torch.logsumexp(x, dim=3)
            w = torch.where(z[..., None] == NEG, 0.0, torch.exp(x - z[..., None]))
            y = torch.matmul(w.reshape(heads, -1, p + n), values).reshape(heads, b - a, group, d) * float(s["v_scale"])
            out[start[r] + a:start[r] + b] = y.permute(1, 0, 2, 3).reshape(b - a, heads * group, d)
            lse[start[r] + a:start[r] + b] = z.permute(1, 0, 2).reshape(b - a, heads * group)
            if scores is not None:
                if a == 0:
                    scores[r, :, :n] *= float(s["decay"])
                scores[r, :, :n] += w[..., p:].sum(dim=(1, 2))
    answer = {"out": out, "lse": lse}
    if scores is not None:
        answer["scores"] = scores
    return answer


def _evict_exact(s):
    cache, heads, bs = s["cache"], s["cache"].shape[3], s["cache"].shape[2]
    scores, positions = s["scores"].cpu().numpy().astype(np.float64), s["positions"].cpu().numpy()
    lens, budget, seen = (s[k].cpu().numpy().astype(np.int64) for k in ("lens", "budget", "seen"))
    table = s["table"].cpu().numpy()
    new_scores, new_positions = np.zeros_like(scores), np.full_like(positions, -1)
    new = np.minimum(lens, np.maximum(budget, 0))
    moves = []
    for r in range(len(lens)):
        n, b = int(lens[r]), int(new[r])
        for h in range(heads):
            x, p = scores[r, h, :n], positions[r, h, :n]
            safe = (p < s["sinks"]) | (p >= seen[r] - s["recent"])
            best = np.lexsort((np.arange(n), -np.where(np.isnan(x), -np.inf, x), ~safe))[:b]
            best.sort()
            come = best[best >= b]
            free = np.setdiff1d(np.arange(b), best, assume_unique=True)
            source = np.arange(b)
            source[free] = come
            new_scores[r, h, :b], new_positions[r, h, :b] = x[source], p[source]
            if len(come):
                moves.append(np.stack([table[r, come // bs], come % bs, table[r, free // bs], free % bs,
                                       np.full(len(come), h)]))
    result = cache.double()
    if moves:
        m = torch.from_numpy(np.concatenate(moves, axis=1).astype(np.int64)).to(cache.device)
        result[m[2], :, m[3], m[4]] = result[m[0], :, m[1], m[4]]
    dev = cache.device
    return {"lens": torch.from_numpy(new.astype(np.int32)).to(dev), "scores": torch.from_numpy(new_scores).to(dev),
            "positions": torch.from_numpy(new_positions).to(dev), "cache": result}
