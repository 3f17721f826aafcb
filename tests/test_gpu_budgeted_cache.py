"""The budgeted cache's loop: a shared prefix, ragged prompts, decode steps and evictions.  Every attention is held to the
definition over the cache as it stands, every eviction is exact."""

import numpy as np
import pytest
import torch

from attention_cases import bounds
from oracle import attention as oracle
from runtime.budgeted_cache import BudgetedCache

HEADS, GROUP, DIM = 2, 3, 64


def check_attend(cache, query, scale, q_start=None, longest=1):
    scores = cache.scores.cpu().numpy()
    shared = cache.prefix_table is not None
    want = oracle.attend(
        query.double().cpu().numpy(), cache.kv.double().cpu().numpy(), cache.table.cpu().numpy(), cache.lens.cpu().numpy(),
        scale, None if q_start is None else q_start.cpu().numpy(), longest,
        cache.prefix_table.cpu().numpy() if shared else None, cache.prefix_len.cpu().numpy() if shared else None, None,
        cache.k_scale, cache.v_scale, scores, cache.decay)
    out, lse = cache.attend(query, scale, q_start, longest)
    out_bound, lse_bound, relative = bounds(want, DIM, query.dtype)
    assert np.all(np.abs(out.double().cpu().numpy() - want["out"]) <= out_bound)
    assert np.all(np.abs(lse.double().cpu().numpy() - want["lse"]) <= lse_bound)
    off = np.abs(cache.scores.double().cpu().numpy() - want["scores"])
    assert np.all(off <= (2 * relative.max() + (longest * GROUP + 8) * 2.0**-24) * np.abs(want["scores"]) + 2.0**-100)


def check_trim(cache):
    before = [x.cpu().numpy() for x in (cache.table, cache.lens, cache.scores, cache.positions)]
    want = oracle.evict(cache.kv.double().cpu().numpy(), *before, [cache.budget] * len(before[1]), cache.seen.cpu().numpy(),
                        cache.recent, cache.sinks)
    cache.trim()
    assert np.array_equal(cache.lens.cpu().numpy(), want["lens"])
    assert np.array_equal(cache.scores.cpu().numpy(), want["scores"])
    assert np.array_equal(cache.positions.cpu().numpy(), want["positions"])
    assert np.array_equal(cache.kv.double().cpu().numpy(), want["cache"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float8_e4m3fn], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("prefix", [0, 37])
def test_prompts_steps_and_evictions(dtype, prefix):
    rows, scale = 5, DIM**-0.5
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    fp8 = dtype == torch.float8_e4m3fn
    cache = BudgetedCache(rows, HEADS, DIM, budget=40, slack=24, prefix=prefix, block=16, dtype=dtype, recent=8, sinks=2,
                          decay=0.75, k_scale=0.02 if fp8 else 1.0, v_scale=0.02 if fp8 else 1.0)
    kind = torch.bfloat16 if fp8 else dtype

    def some(n, heads):
        return torch.randn(n, heads, DIM, generator=gen, device="cuda")

    def new(n):
        part = some(n, HEADS) / cache.k_scale
        return part, part.flip(0) + 0.5 / cache.v_scale

    if prefix:
        cache.set_prefix(*new(prefix))
    start = torch.tensor([0, 30, 30, 64, 65, 107], dtype=torch.int32, device="cuda")
    cache.append(*new(107), start, 42)
    check_attend(cache, (1.5 * some(107, HEADS * GROUP)).to(kind), scale, start, 42)
    trims = 0
    for _ in range(50):
        cache.append(*new(rows))
        check_attend(cache, (1.5 * some(rows, HEADS * GROUP)).to(kind), scale)
        if cache.full:
            check_trim(cache)
            trims += 1
    assert trims == 2 and cache.lens.max() == 50 - 22 - 24 + 40
    assert cache.seen.tolist() == [80, 50, 84, 51, 92]
    # what a row holds: distinct positions, the first and the newest among them
    for r in range(rows):
        n = int(cache.lens[r])
        for h in range(HEADS):
            held = sorted(cache.positions[r, h, :n].tolist())
            assert len(set(held)) == n and held[0] == 0 and held[1] == 1
            assert held[-8:] == list(range(int(cache.seen[r]) - 8, int(cache.seen[r])))


def test_refusals():
    with pytest.raises(ValueError, match="budget"):
        BudgetedCache(2, HEADS, DIM, budget=0, device="cpu")
    cache = BudgetedCache(2, HEADS, DIM, budget=4, slack=2, prefix=3, device="cpu")
    rows = torch.zeros(2, HEADS, DIM)
    for _ in range(6):
        assert not cache.full
        cache.append(rows, rows)
    assert cache.full
    with pytest.raises(ValueError, match="trim"):
        cache.append(rows, rows)
    with pytest.raises(ValueError, match="prefix"):
        cache.set_prefix(torch.zeros(17, HEADS, DIM), torch.zeros(17, HEADS, DIM))
    with pytest.raises(ValueError, match="prefix"):
        BudgetedCache(2, HEADS, DIM, budget=4, device="cpu").set_prefix(rows, rows)
    with pytest.raises(ValueError, match="device tensor"):
        cache.attend(torch.zeros(2, HEADS, DIM, dtype=torch.bfloat16), 0.1)


def test_append_places_tokens():
    cache = BudgetedCache(2, 1, 32, budget=20, slack=4, block=8, dtype=torch.float32, device="cpu")
    start = torch.tensor([0, 3, 12], dtype=torch.int32)
    rows = torch.arange(12.0).view(12, 1, 1).expand(12, 1, 32)
    cache.append(rows, -rows, start, 9)
    cache.append(100 + rows[:2], rows[:2])
    assert cache.lens.tolist() == [4, 10] and cache.seen.tolist() == [4, 10] and cache.longest == 10
    flat = cache.kv[cache.table.long()].permute(0, 2, 1, 3, 4, 5).reshape(2, 2, 24, 32)[..., 0]
    assert flat[0, 0, :4].tolist() == [0, 1, 2, 100] and flat[0, 1, :4].tolist() == [0, -1, -2, 0]
    assert flat[1, 0, :10].tolist() == [3, 4, 5, 6, 7, 8, 9, 10, 11, 101]
    assert cache.positions[1, 0, :11].tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, -1]
