"""Paged batches for the attention and eviction tests, and the bounds their results are held to."""

from __future__ import annotations

import numpy as np
import torch

from oracle import attention as oracle

QUERY_TYPE = {torch.float32: torch.float32, torch.float16: torch.float16, torch.bfloat16: torch.bfloat16,
              torch.float8_e4m3fn: torch.bfloat16}


class Batch:
    """Rows of ``lens`` own tokens, ``counts`` queries each, behind prefixes of ``prefixes`` tokens whose rows end
    at ``borders``; ``spare`` pages at the end of the pool belong to nobody."""

    def __init__(self, lens, counts=None, prefixes=(), borders=None, heads=2, group=4, dim=64, block=16,
                 dtype=torch.bfloat16, seed=0, spare=2, spread=1.5):
        rng = np.random.default_rng(seed)
        rows = len(lens)
        self.dtype, self.block, self.heads, self.group, self.dim = dtype, block, heads, group, dim
        self.lens = np.asarray(lens, np.int32)
        self.counts = None if counts is None else np.asarray(counts)
        tokens = rows if counts is None else int(self.counts.sum())
        self.q_start = None if counts is None else np.concatenate([[0], np.cumsum(self.counts)]).astype(np.int32)
        self.max_query = 1 if counts is None else max(1, int(self.counts.max(initial=1)))
        need = -(-self.lens.astype(np.int64) // block)
        pneed = -(-np.asarray(prefixes, np.int64) // block)
        pool = int(need.sum() + pneed.sum()) + 1 + spare
        ids = rng.permutation(np.arange(1, pool - spare)).astype(np.int32)
        self.table = np.full((rows, max(1, int(need.max(initial=0)) + 1)), 2**31 - 1, np.int32)  # past a row: anything
        at = 0
        for r in range(rows):
            self.table[r, : need[r]] = ids[at : at + need[r]]
            at += need[r]
        self.prefix_table = self.prefix_lens = self.prefix_rows = None
        if len(prefixes):
            self.prefix_lens = np.asarray(prefixes, np.int32)
            self.prefix_table = np.full((len(prefixes), max(1, int(pneed.max()))), -7, np.int32)
            for g in range(len(prefixes)):
                self.prefix_table[g, : pneed[g]] = ids[at : at + pneed[g]]
                at += pneed[g]
            if borders is not None:
                self.prefix_rows = np.asarray(borders, np.int32)
        qtype = QUERY_TYPE[dtype]
        self.k_scale = self.v_scale = 1.0
        raw = rng.standard_normal((pool, 2, block, heads, dim))
        raw[:, 1] += 0.5
        if dtype == torch.float8_e4m3fn:
            self.k_scale, self.v_scale = 0.02, 0.015
            raw /= 0.02
        self.cache = torch.from_numpy(raw).float().to(dtype)
        self.query = torch.from_numpy(spread * rng.standard_normal((tokens, heads * group, dim))).float().to(qtype)
        self.scale = dim**-0.5
        self.scores = None
        self.decay = 1.0

    def with_scores(self, seed=1, decay=0.75):
        rng = np.random.default_rng(seed)
        self.scores = torch.from_numpy(
            rng.exponential(1.0, (len(self.lens), self.heads, self.table.shape[1] * self.block))).float()
        self.decay = decay
        return self

    def want(self):
        return oracle.attend(
            self.query.double().numpy(), self.cache.double().numpy(), self.table, self.lens, self.scale, self.q_start,
            self.max_query, self.prefix_table, self.prefix_lens, self.prefix_rows, self.k_scale, self.v_scale,
            None if self.scores is None else self.scores.numpy(), self.decay)

    def on_gpu(self):
        def up(x):
            return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()

        return dict(query=self.query.cuda(), kv_cache=self.cache.cuda(), table=up(self.table), lens=up(self.lens),
                    scale=self.scale, q_start=up(self.q_start), max_query=self.max_query,
                    prefix_table=up(self.prefix_table), prefix_lens=up(self.prefix_lens),
                    prefix_rows=up(self.prefix_rows), k_scale=self.k_scale, v_scale=self.v_scale,
                    scores=None if self.scores is None else self.scores.cuda(), decay=self.decay)


def bounds(want, dim, qtype):
    """How far a float32 computation may be off the definition: per query, from the sizes alone.

    u = 2^-24.  A logit is a sum of ``dim`` products in float32, scaled: off by at most (dim + 4) u of the sum
    of its terms' magnitudes (``reach``).  A weight exp(s - lse) is then off by a relative 2 (dim + 4) u reach,
    once from its own logit and once from the sum's, plus the sum over ``keys`` terms, the exponential and the
    joining of chunks: (keys + 64) u.  For 16-bit outputs the weights may be rounded to the type before they
    meet the values (half a step each), and the result is rounded to it."""
    u = 2.0**-24
    relative = 2 * (dim + 4) * u * want["reach"] + (want["keys"] + 64) * u
    half = 0.0 if qtype == torch.float32 else torch.finfo(qtype).eps / 2
    out = (relative + half)[..., None] * want["weighed"] + max(half, u) * np.abs(want["out"])
    # the smallest steps of the type, where its values are subnormal
    out = out + torch.finfo(qtype).tiny * torch.finfo(qtype).eps
    finite = np.where(np.isfinite(want["lse"]), want["lse"], 0.0)
    lse = relative + 4 * u * np.abs(finite)
    return out, lse, relative


def check(batch, out, lse, scores=None, want=None):
    want = batch.want() if want is None else want
    out_bound, lse_bound, relative = bounds(want, batch.dim, batch.query.dtype)
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.array_equal(np.isneginf(got_lse), np.isneginf(want["lse"]))
    assert np.all(np.isfinite(got)), "out is not finite"
    dead = np.isneginf(want["lse"])
    assert np.all(got[dead] == 0)
    over = np.abs(got - want["out"]) - out_bound
    assert over.max(initial=-1.0) <= 0, f"out off by {np.abs(got - want['out']).max()}"
    gap = np.where(dead, 0.0, np.abs(np.where(dead, 0.0, got_lse) - np.where(dead, 0.0, want["lse"])))
    assert np.all(gap <= lse_bound), f"lse off by {gap.max()}"
    if scores is not None:
        # a score adds one weight per query row of its head: each off by `relative`, their sum by u a term
        queries = batch.max_query * batch.group
        rel = (2 * relative.max(initial=0.0) + (queries + 8) * 2.0**-24)
        tolerance = rel * np.abs(want["scores"]) + 2.0**-100
        off = np.abs(scores.double().cpu().numpy() - want["scores"])
        assert np.all(off <= tolerance), f"scores off by {off.max()}"
