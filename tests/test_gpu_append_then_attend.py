"""Tokens appended with advancing counts and then attended to, rows that bring more than max_query among them: a kept token
sees itself and every slot before it, and nothing that was not kept."""

import numpy as np
import pytest
import torch

from attention_cases import Batch, bounds
from oracle import attention as oracle
from runtime.append import append_tokens
from runtime.budgeted_cache import BudgetedCache
from runtime.prefix_attention import prefix_attention

pytestmark = pytest.mark.gpu
F32, F16, BF16, FP8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


def kept_tokens(start, max_query):
    """Which tokens are kept, and the starts that the kept ones alone have."""
    counts = np.minimum(np.diff(start), max_query)
    token = np.concatenate([np.arange(a, a + n) for a, n in zip(start, counts)]).astype(int)
    return token, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def check(query, cache, table, lens, scale, start, max_query, prefix_table, prefix_lens, k_scale, v_scale, scores, decay, got):
    """``got`` (out, lse, scores) against the attention of the kept tokens alone."""
    token, alone = kept_tokens(start, max_query)
    want = oracle.attend(query.double().cpu().numpy()[token], cache.double().cpu().numpy(), table.cpu().numpy(),
                         lens.cpu().numpy(), scale, alone, max_query, prefix_table, prefix_lens, None, k_scale, v_scale,
                         scores, decay)
    out, lse, new = (x.double().cpu().numpy() for x in got)
    none = np.ones(len(out), bool)
    none[token] = False
    assert np.all(out[none] == 0) and np.all(np.isneginf(lse[none]))
    out_bound, lse_bound, relative = bounds(want, query.shape[2], query.dtype)
    dead = np.isneginf(want["lse"])
    assert np.array_equal(np.isneginf(lse[token]), dead)
    assert np.all(np.abs(out[token] - want["out"]) <= out_bound)
    assert np.all(np.abs(np.where(dead, 0, lse[token]) - np.where(dead, 0, want["lse"])) <= lse_bound)
    group = query.shape[1] // cache.shape[3]
    off = np.abs(new - want["scores"])
    assert np.all(off <= (2 * relative.max(initial=0.0) + (max_query * group + 8) * 2.0**-24) * np.abs(want["scores"]) + 2.0**-100)


@pytest.mark.parametrize("dtype", [BF16, F16, F32, FP8], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("prefix", [0, 37])
@pytest.mark.parametrize("group,most,counts", [
    (3, 6, [9, 30, 0, 5]),  # few queries, their logits kept
    (2, 9, [40, 3, 10, 9]),
    (4, 70, [90, 300, 0, 70]),  # tiles of prompt chunks
    (8, 130, [131, 1, 200]),
])
def test_budgeted_cache(dtype, prefix, group, most, counts):
    heads, dim, rows = 2, 64, len(counts)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(11)
    fp8 = dtype == FP8
    kind = BF16 if fp8 else dtype
    cache = BudgetedCache(rows, heads, dim, budget=2 * most, slack=most, prefix=prefix, block=16, dtype=dtype, decay=0.75,
                          k_scale=0.02 if fp8 else 1.0, v_scale=0.02 if fp8 else 1.0)

    def new(n, h):
        return torch.randn(n, h, dim, generator=gen, device="cuda")

    if prefix:
        cache.set_prefix(new(prefix, heads) / cache.k_scale, new(prefix, heads) / cache.v_scale)
    scale = dim**-0.5
    for step in (counts, counts[::-1]):
        start = np.concatenate([[0], np.cumsum(step)]) + 3  # padded on both sides
        n = int(start[-1]) + 2
        starts = torch.from_numpy(start.astype(np.int32)).cuda()
        cache.append(new(n, heads) / cache.k_scale, new(n, heads) / cache.v_scale, starts, most)
        query = (1.5 * new(n, heads * group)).to(kind)
        before = cache.scores.cpu().numpy().astype(np.float64)
        out, lse = cache.attend(query, scale, starts, most)
        check(query, cache.kv, cache.table, cache.lens, scale, start, most, cache.prefix_table.cpu().numpy() if prefix else None,
              cache.prefix_len.cpu().numpy() if prefix else None, cache.k_scale, cache.v_scale, before, cache.decay,
              (out, lse, cache.scores))


@pytest.mark.parametrize("dtype", [BF16, F32, FP8], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("lens,counts,most,prefixes", [
    ([40, 7, 90], [9, 2, 30], 5, []),
    ([140, 7, 90], [9, 2, 30], 5, [33]),
    ([400, 170, 290], [300, 2, 160], 100, []),
    ([400, 170, 1290], [300, 2, 160], 100, [70]),
    ([700], [900], 600, []),
    ([64] * 40, [5] * 40, 3, [2000]),  # few queries a row behind a prefix read for all of them
])
def test_lengths_of_kept_tokens(dtype, lens, counts, most, prefixes):
    b = Batch(lens, counts, prefixes=prefixes, heads=2, group=4, dim=64, dtype=dtype, seed=3).with_scores()
    b.max_query = most
    args = b.on_gpu()
    out, lse = prefix_attention(**args, kept=most)
    check(b.query, b.cache, torch.from_numpy(b.table), torch.from_numpy(b.lens), b.scale, b.q_start, most, b.prefix_table,
          b.prefix_lens, b.k_scale, b.v_scale, b.scores.numpy(), b.decay, (out, lse, args["scores"]))
    # rows within max_query: the same bits with it and without
    b = Batch(lens, counts, prefixes=prefixes, heads=2, group=4, dim=64, dtype=dtype, seed=4).with_scores()
    first, second = b.on_gpu(), b.on_gpu()
    one, two = prefix_attention(**first), prefix_attention(**second, kept=b.max_query)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1]) and torch.equal(first["scores"], second["scores"])


def test_bounds_of_their_own():
    """Two appends attended to at once, and fewer queries than were appended: each query sees what it did before."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(4)
    x = torch.randn(16, 8, 64, generator=gen, device="cuda").to(BF16)
    keys, values, query = x[:, :2], x[:, 2:4], x[:, 4:]
    start = torch.tensor([0, 8, 16], dtype=torch.int32, device="cuda")

    def cache():
        return BudgetedCache(2, 2, 64, budget=32, slack=8)

    whole = cache()
    whole.append(keys, values, start, 8)
    want = whole.attend(query, 0.125, start, 8)
    pieces = cache()
    for part in (slice(0, 4), slice(4, 8)):
        both = torch.cat([keys[part], keys[8:][part]]), torch.cat([values[part], values[8:][part]])
        pieces.append(*both, torch.tensor([0, 4, 8], dtype=torch.int32, device="cuda"), 4)
    got = pieces.attend(query, 0.125, start, 8)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    again = cache()
    again.append(keys, values, start, 8)
    out, lse = again.attend(query, 0.125, start, 3)
    first = torch.tensor([0, 1, 2, 8, 9, 10], device="cuda")
    assert torch.allclose(out[first].float(), want[0][first].float(), rtol=2.0**-7, atol=2.0**-7)
    assert torch.allclose(lse[first], want[1][first], rtol=1e-4, atol=1e-4)
    none = torch.ones(16, dtype=torch.bool, device="cuda")
    none[first] = False
    assert not out[none].any() and torch.isneginf(lse[none]).all()


def test_the_public_calls_together():
    """append_tokens with advance, then prefix_attention of the same starts and max_query."""
    heads, group, dim, block, most = 2, 3, 64, 16, 4
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    start = np.array([0, 9, 9, 13, 14])
    starts = torch.from_numpy(start.astype(np.int32)).cuda()
    cache = torch.randn(21, 2, block, heads, dim, generator=gen, device="cuda").to(BF16)
    table = torch.arange(1, 21, dtype=torch.int32, device="cuda").view(4, 5)
    lens = torch.tensor([30, 7, 16, 0], dtype=torch.int32, device="cuda")
    x = torch.randn(14, heads * (group + 2), dim, generator=gen, device="cuda").to(BF16)
    query, keys, values = x.split([heads * group, heads, heads], 1)
    scores = torch.zeros(4, heads, 80, device="cuda")
    append_tokens(cache, table, lens, keys, values, q_start=starts, max_query=most, scores=scores, advance=True)
    assert lens.tolist() == [34, 7, 20, 1]
    out, lse = prefix_attention(query, cache, table, lens, 0.125, q_start=starts, max_query=most, scores=scores, kept=most)
    check(query, cache, table, lens, 0.125, start, most, None, None, 1.0, 1.0, np.zeros((4, heads, 80)), 1.0, (out, lse, scores))
