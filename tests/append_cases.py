"""Batches of new tokens for the append and rotation tests, and the bounds their results are held to."""

from __future__ import annotations

import numpy as np
import torch

from oracle import append as oracle


def bound(want, reach, dtype, dim, normed, angle, scaled=True):
    """How far a float32 computation rounded once to ``dtype`` may be off ``want``, from the sizes alone.

    u = 2^-24.  The sum of ``dim`` squares is off by a relative (dim + 2) u, half of that in its root, and the root, its
    product with the element, the weight and that product add 8 u.  A cosine is off by pi u for its angle's rounding to a
    fraction of a turn (at most half a turn), by 2^-51 of the largest angle for the float64 products before, by 4 u of the
    function's own and u of the scale; a rotated element sums two products, 3 u, of magnitudes ``reach``.  The cache's scale
    is a rounded reciprocal and a product: 2 u.  The result is rounded once, by half a step relative to the value, or half
    the least step of the type's subnormals."""
    u = 2.0**-24
    relative = (dim / 2 + 9) * u * normed + (3.15 + 4 + 1 + 3) * u + angle * 2.0**-51 + 2 * u * scaled
    off = relative * reach
    info = torch.finfo(dtype)
    if dtype == torch.float32:
        return off + u * np.abs(want) + info.tiny
    least = 2.0**-10 if dtype == torch.float8_e4m3fn else info.tiny * info.eps / 2
    return off + info.eps / 2 * (np.abs(want) + off) + least


class Tokens:
    """New tokens of rows of ``lens`` tokens, ``counts`` new ones each (None: one a row), ``ahead`` and ``behind`` tokens of
    no row around them; ``spare`` pages at the end of the pool belong to nobody.  With ``advance`` the lengths are those
    before the call."""

    def __init__(self, lens, counts=None, q_heads=8, kv_heads=2, dim=64, pairs=None, block=16, dtype=torch.bfloat16, kv=None,
                 adjacent=False, norm=None, axes=0, evicting=False, advance=False, ahead=0, behind=0, max_query=None,
                 first=False, seed=0, spare=2, far=0, width=None, offset=0.0, scale=1.0, no_query=False, weight_type=None):
        rng = np.random.default_rng(seed)
        rows = len(lens)
        self.dtype, self.kv, self.dim, self.block = dtype, dtype if kv is None else kv, dim, block
        self.kv_heads, self.q_heads, self.adjacent, self.advance = kv_heads, q_heads, adjacent, advance
        self.lens = np.asarray(lens, np.int32)
        self.counts = np.ones(rows, int) if counts is None else np.asarray(counts)
        tokens = int(self.counts.sum()) + ahead + behind
        self.q_start = None
        if counts is not None or ahead or behind:
            self.q_start = (np.concatenate([[0], np.cumsum(self.counts)]) + ahead).astype(np.int32)
        self.max_query = max_query or max(1, int(self.counts.max(initial=1)))
        after = self.lens.astype(np.int64) + (self.counts if advance else 0)
        need = -(-after // block)
        pool = int(need.sum()) + 1 + spare
        ids = rng.permutation(np.arange(1, pool - spare)).astype(np.int32)
        width = max(1, int(need.max(initial=0)) + 1) if width is None else width
        self.table = np.full((rows, width), 2**31 - 1, np.int32)  # past a row: anything
        at = 0
        for r in range(rows):
            m = min(need[r], width)
            self.table[r, :m] = ids[at:at + m]
            at += need[r]
        packed = rng.standard_normal((tokens, q_heads + 2 * kv_heads, dim))
        packed[:, q_heads + kv_heads:] += 0.5
        self.packed = torch.from_numpy(packed).float().to(dtype)
        fp8 = self.kv == torch.float8_e4m3fn
        self.k_scale, self.v_scale = (0.02, 0.015) if fp8 else (1.0, 1.0)
        raw = rng.standard_normal((pool, 2, block, kv_heads, dim)) / self.k_scale
        self.cache = torch.from_numpy(raw).float().clamp(-448 if fp8 else None, 448 if fp8 else None).to(self.kv) if fp8 \
            else torch.from_numpy(raw).float().to(self.kv)
        pairs = dim // 2 if pairs is None else pairs
        self.frequencies = 10000.0 ** -(np.arange(pairs) / max(1, pairs)) if pairs else None
        self.axes = self.positions = self.q_weight = self.k_weight = None
        if axes:
            self.axes = rng.integers(0, axes, size=pairs).astype(np.int32)
            self.positions = rng.integers(0, far or 5000, size=(axes, tokens)).astype(np.int32)
        if norm:
            kind = weight_type or dtype
            shapes = ((q_heads, dim), (kv_heads, dim)) if norm == "heads" else ((dim,), (dim,))
            self.q_weight, self.k_weight = (
                torch.from_numpy(1 - offset + 0.3 * rng.standard_normal(shape)).float().to(kind) for shape in shapes)
        self.offset, self.scale, self.eps, self.no_query = offset, scale, 1e-6, no_query
        self.seen = self.scores = self.slot_positions = self.first = None
        if evicting:
            self.seen = (self.lens + rng.integers(0, far or 3000, size=rows)).astype(np.int32)
            shape = (rows, kv_heads, width * block + 3)
            self.scores = rng.exponential(1.0, shape).astype(np.float32)
            self.slot_positions = rng.integers(0, 3000, size=shape).astype(np.int32)
        if first:
            self.first = rng.integers(0, 3000, size=rows).astype(np.int32)

    def parts(self, packed):
        q, k = self.q_heads, self.q_heads + self.kv_heads
        return packed[:, :q], packed[:, q:k], packed[:, k:]

    def want(self):
        query, keys, values = self.parts(self.packed.double().numpy())
        double = [None if w is None else w.double().numpy() for w in (self.q_weight, self.k_weight)]
        return oracle.append(
            self.cache.double().numpy(), self.table, self.lens, keys, values, self.q_start, self.max_query,
            None if self.no_query else query, self.positions, self.frequencies, self.axes, self.adjacent, self.scale, *double,
            self.eps, self.offset, self.k_scale, self.v_scale, self.seen, self.first, self.scores, self.slot_positions,
            self.advance)

    def on_gpu(self):
        def up(x):
            return None if x is None else x.cuda() if isinstance(x, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(x)).cuda()

        query, keys, values = self.parts(self.packed.cuda())
        return dict(kv_cache=self.cache.cuda(), table=up(self.table), lens=up(self.lens), keys=keys, values=values,
                    q_start=up(self.q_start), max_query=self.max_query, query=None if self.no_query else query,
                    positions=up(self.positions), frequencies=up(self.frequencies), axes=up(self.axes),
                    adjacent=self.adjacent, rotary_scale=self.scale, q_weight=None if self.no_query else up(self.q_weight),
                    k_weight=up(self.k_weight), eps=self.eps, weight_offset=self.offset, k_scale=self.k_scale,
                    v_scale=self.v_scale, seen=up(self.seen), first=up(self.first), scores=up(self.scores),
                    slot_positions=up(self.slot_positions), advance=self.advance)

    def angle(self, want):
        """The largest angle, in radians."""
        if self.frequencies is None:
            return 0.0
        if self.positions is not None:
            return float(np.abs(self.positions).max(initial=0))
        top = np.abs(self.lens.astype(np.int64) if self.seen is None else self.seen.astype(np.int64)).max(initial=0)
        return float(top + self.counts.max(initial=0) + (0 if self.first is None else self.first.max(initial=0)))


def check(batch, args, query, want=None):
    """Everything the call wrote against the definition, everything else as it was."""
    want = batch.want() if want is None else want
    normed, angle = batch.k_weight is not None, batch.angle(want)
    cache = args["kv_cache"].cpu()
    got, wrote = cache.double().numpy(), want["wrote"]
    same = batch.cache.view(torch.uint8).numpy() == cache.view(torch.uint8).numpy()
    same = same.reshape(*batch.cache.shape, -1).all(axis=-1)
    assert np.all(same[~wrote]), "a slot that no token has changed"
    limit = bound(want["cache"], want["reach"], batch.kv, batch.dim, normed, angle)
    off = np.abs(np.where(wrote, got - want["cache"], 0.0))
    assert np.all(np.isfinite(got[wrote]))
    assert np.all(off <= limit), f"cache off by {off.max()}"
    if want["query"] is not None:
        mine = query.double().cpu().numpy()
        limit = bound(want["query"], want["query_reach"], batch.dtype, batch.dim, normed, angle, False)
        off = np.abs(mine - want["query"])
        assert np.all(off <= limit), f"query off by {off.max()}"
        assert np.all(mine[want["query_reach"].sum(axis=(1, 2)) == 0] == 0)
    else:
        assert query is None
    assert np.array_equal(args["lens"].cpu().numpy(), want["lens"])
    for name in ("seen", "scores", "slot_positions"):
        if want[name] is not None:
            assert np.array_equal(args[name].cpu().numpy(), want[name]), name
