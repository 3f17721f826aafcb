"""What BudgetedCache.append takes and refuses, on the host: padding around the rows' tokens, rows past max_query, and
counts of tokens that are not the rows'."""

import pytest
import torch

from runtime.budgeted_cache import BudgetedCache

ROWS, HEADS, DIM, BLOCK = 3, 2, 32, 4


def cache_of(budget=8, slack=4):
    return BudgetedCache(ROWS, HEADS, DIM, budget=budget, slack=slack, block=BLOCK, dtype=torch.float32, device="cpu")


def tokens(n, first=1.0):
    rows = torch.arange(first, first + n).view(n, 1, 1).expand(n, HEADS, DIM)
    return rows, -rows


def held(cache):
    """The first element of each row's keys, by slot."""
    flat = cache.kv[cache.table.long(), 0]  # [rows, width, block, heads, dim]
    return flat.reshape(ROWS, -1, HEADS, DIM)[:, :, 0, 0]


def expect(cache, lens, rows):
    assert cache.lens.tolist() == lens and cache.seen.tolist() == lens
    assert cache.longest >= max(lens)
    for r, want in enumerate(rows):
        assert held(cache)[r].tolist() == want + [0.0] * (held(cache).shape[1] - len(want))
        for h in range(HEADS):
            assert cache.positions[r, h].tolist() == list(range(lens[r])) + [-1] * (cache.positions.shape[2] - lens[r])
    assert torch.all(cache.scores == 5.0)  # of kept tokens cleared: the caller set it again


def fill_scores(cache):
    for r in range(ROWS):
        n = int(cache.lens[r])
        assert torch.all(cache.scores[r, :, :n] == 0.0)  # a new token starts at 0
        cache.scores[r, :, :n] = 5.0


@pytest.mark.parametrize("ahead,behind", [(0, 2), (2, 0), (3, 5)])
def test_tokens_of_no_row(ahead, behind):
    cache = cache_of()
    cache.scores.fill_(5.0)
    start = torch.tensor([0, 2, 2, 5], dtype=torch.int32) + ahead
    cache.append(*tokens(5 + ahead + behind), start, 3)
    fill_scores(cache)
    expect(cache, [2, 0, 3], [[1.0 + ahead, 2.0 + ahead], [], [3.0 + ahead, 4.0 + ahead, 5.0 + ahead]])


def test_rows_past_max_query():
    cache = cache_of()
    cache.scores.fill_(5.0)
    cache.append(*tokens(15), torch.tensor([0, 13, 14, 15], dtype=torch.int32), 12)
    fill_scores(cache)
    expect(cache, [12, 1, 1], [[float(x) for x in range(1, 13)], [14.0], [15.0]])
    assert cache.full
    with pytest.raises(ValueError, match="trim"):
        cache.append(*tokens(ROWS))


def test_the_default_bound_is_one_token():
    cache = cache_of()
    cache.scores.fill_(5.0)
    cache.append(*tokens(5), torch.tensor([0, 3, 3, 5], dtype=torch.int32))
    fill_scores(cache)
    expect(cache, [1, 0, 1], [[1.0], [], [4.0]])


def test_starts_past_the_tokens():
    cache = cache_of()
    cache.scores.fill_(5.0)
    cache.append(*tokens(3), torch.tensor([0, 2, 4, 9], dtype=torch.int32), 4)  # the second row has one, the third none
    fill_scores(cache)
    expect(cache, [2, 1, 0], [[1.0, 2.0], [3.0], []])


def test_padding_beside_full_rows():
    cache = cache_of(budget=4, slack=4)
    cache.append(*tokens(24), torch.tensor([0, 8, 16, 24], dtype=torch.int32), 8)
    before = held(cache).clone()
    cache.longest = 0  # as if the host knew of room
    with pytest.raises(ValueError, match="trim"):
        cache.append(*tokens(9), torch.tensor([0, 0, 0, 0], dtype=torch.int32), 9)
    cache.append(*tokens(4), torch.tensor([2, 2, 2, 2], dtype=torch.int32), 2)
    assert torch.equal(held(cache), before) and cache.lens.tolist() == [8, 8, 8]


def test_refusals():
    cache = cache_of()
    k, v = tokens(ROWS)
    for n in (0, 2, 4):
        with pytest.raises(ValueError, match="q_start"):
            cache.append(*tokens(n))
    with pytest.raises(ValueError, match="q_start"):
        cache.append(k, v, torch.tensor([0, 1, 3], dtype=torch.int32), 2)
    with pytest.raises(ValueError, match="values"):
        cache.append(k, v[:2])
    with pytest.raises(ValueError, match="keys"):
        cache.append(k[:, :1], v[:, :1])
    with pytest.raises(ValueError, match="keys"):
        cache.append(k[..., :1], v[..., :1])
    with pytest.raises(ValueError, match="tokens a row"):
        cache.append(k, v, torch.tensor([0, 1, 2, 3], dtype=torch.int32), 0)
    with pytest.raises(ValueError, match="keys"):
        BudgetedCache(ROWS, HEADS, DIM, budget=4, prefix=8, device="cpu").set_prefix(k[:, :1], v[:, :1])
    assert cache.lens.tolist() == [0, 0, 0] and cache.longest == 0
