"""Token eviction against its definition, token by token: what stays, where it goes, the cache, scores, positions
and lengths, all exact."""

import numpy as np
import pytest
import torch

from oracle import attention as oracle
from runtime.eviction import evict_tokens

pytestmark = pytest.mark.gpu


def batch(lens, heads=2, dim=32, block=16, dtype=torch.bfloat16, seed=0, ties=False, room=1):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, np.int32)
    need = -(-lens.astype(np.int64) // block)
    width = int(need.max(initial=0)) + room
    pool = int(need.sum()) + 3
    ids = rng.permutation(np.arange(1, pool)).astype(np.int32)
    table = np.full((len(lens), width), -1, np.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = ids[at : at + n]
        at += n
    capacity = width * block
    scores = rng.exponential(1.0, (len(lens), heads, capacity)).astype(np.float32)
    if ties:
        scores = np.floor(scores * 2)
        scores[scores == 1] *= rng.choice([-0.0, 1.0], size=(scores == 1).sum())
    positions = np.tile(np.arange(capacity, dtype=np.int32), (len(lens), heads, 1))
    cache = torch.from_numpy(rng.standard_normal((pool, 2, block, heads, dim)) * 4).float().to(dtype)
    return cache, table, lens, scores, positions


def run(b, budget, seen, in_place=False, fixed=None, **more):
    cache, table, lens, scores, positions = b
    gpu = [cache.cuda(), *(torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (table, lens, scores, positions))]
    want = oracle.evict(cache.double().numpy(), table, lens, scores, positions, budget, seen, **more)
    if in_place:
        more.update(new_scores=gpu[3], new_positions=gpu[4])
    limit = fixed if fixed is not None else torch.tensor(budget, dtype=torch.int32).cuda()
    got = evict_tokens(*gpu, limit, torch.tensor(seen, dtype=torch.int32).cuda(), **more)
    torch.cuda.synchronize()
    assert np.array_equal(got[0].cpu().numpy(), want["lens"])
    assert np.array_equal(got[1].cpu().numpy(), want["scores"], equal_nan=True)
    assert np.array_equal(got[2].cpu().numpy(), want["positions"])
    assert np.array_equal(gpu[0].double().cpu().numpy(), want["cache"])
    if not in_place:
        assert np.array_equal(gpu[3].cpu().numpy(), scores, equal_nan=True)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("ties", [False, True])
def test_lengths_and_budgets(ties, in_place):
    lens = [0, 1, 2, 31, 32, 33, 64, 100, 511, 512, 513, 1500]
    b = batch(lens, ties=ties, seed=1)
    for budget in ([0] * 12, [1] * 12, [16] * 12, [n // 2 for n in lens], [max(0, n - 3) for n in lens],
                   [5000, -4, 2, 7, 31, 32, 63, 99, 500, 511, 512, 1499]):
        run(b, budget, lens, in_place)
        run(b, budget, lens, in_place, recent=10, sinks=3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn],
                         ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_types(dtype, dim):
    run(batch([90, 300], dim=dim, dtype=dtype, seed=dim), [41, 128], [90, 300], recent=8, sinks=4)


@pytest.mark.parametrize("block", [1, 8, 24, 64])
def test_block_sizes(block):
    run(batch([90, 300, 7], heads=3, block=block, seed=block), [41, 128, 3], [90, 300, 7], recent=8, sinks=4)


def test_more_protected_than_the_budget():
    run(batch([200, 50], seed=2), [20, 30], [200, 50], recent=100, sinks=40)
    run(batch([200, 50], seed=2), [20, 30], [200, 50], sinks=10**6)  # everything is
    run(batch([200, 50], seed=2), [20, 30], [2**31 - 1, -(2**31)], recent=2**31 - 1)


def test_special_scores():
    b = batch([300, 300], seed=3)
    rng = np.random.default_rng(5)
    b[3][:] = rng.choice([np.nan, -np.inf, np.inf, -0.0, 0.0, 1e-45, -1e-45, 3e38, 1.0], size=b[3].shape)
    for budget in (10, 77, 150, 299):
        run(b, [budget] * 2, [300] * 2)


def test_one_budget_for_every_row():
    run(batch([90, 300, 20], seed=4), [64] * 3, [90, 300, 20], fixed=64, recent=4)


def test_positions_after_earlier_evictions():
    b = batch([120, 260], seed=6)
    rng = np.random.default_rng(6)
    for r, n in enumerate(b[2]):
        for h in range(2):
            b[4][r, h, :n] = rng.permutation(1000)[:n]
    run(b, [60, 200], [1000, 900], recent=200, sinks=50)


def test_bad_pages_are_left_alone():
    b = batch([100, 64], seed=7)
    b[1][0, 1], b[1][0, 5], b[1][1, 3] = -1, b[0].shape[0], 2**31 - 1
    run(b, [50, 30], [100, 64])


def test_long_rows():
    run(batch([20000, 33000], heads=1, seed=8, ties=True), [9000, 32000], [20000, 33000], recent=64, sinks=4)


def test_strided_buffers_and_offsets_past_32_bits():
    pages, block, heads, dim = 41000, 16, 8, 256
    big = torch.zeros(pages, 2, block, heads, dim, dtype=torch.bfloat16, device="cuda")  # 2.7e9 elements
    cache, table, lens, scores, positions = batch([70, 200], heads=heads, dim=dim, seed=9)
    n = cache.shape[0]
    big[pages - n:] = cache.cuda()
    want = oracle.evict(cache.double().numpy(), table, lens, scores, positions, [33, 90], lens, recent=5)
    moved = torch.from_numpy(np.where(table >= 0, table + pages - n, table)).cuda()
    wide = torch.full((2, heads, scores.shape[2] + 7), 5.0, device="cuda")
    wide[:, :, : scores.shape[2]] = torch.from_numpy(scores)
    target = torch.full((2, heads, scores.shape[2] + 3), 5.0, device="cuda")
    lens_t = torch.from_numpy(lens).cuda()
    got = evict_tokens(big, moved, lens_t, wide[:, :, : scores.shape[2]], torch.from_numpy(positions).cuda(),
                       torch.tensor([33, 90], dtype=torch.int32).cuda(), lens_t, recent=5,
                       new_scores=target[:, :, : scores.shape[2]])
    assert np.array_equal(got[1].cpu().numpy(), want["scores"]) and (target[:, :, scores.shape[2]:] == 5).all()
    assert np.array_equal(big[pages - n:].double().cpu().numpy(), want["cache"])
    assert not big[: pages - n].any()


def test_graph_replays():
    cache, table, lens, scores, positions = batch([120, 260, 40], seed=10)
    want = oracle.evict(cache.double().numpy(), table, lens, scores, positions, [64] * 3, lens)
    up = [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (table, lens, scores, positions)]
    kv, seen = cache.cuda(), torch.from_numpy(lens).cuda()
    out = [torch.empty_like(up[1]), torch.empty_like(up[2]), torch.empty_like(up[3])]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            evict_tokens(kv, *up, 64, seen, new_lens=out[0], new_scores=out[1], new_positions=out[2])
    for _ in range(3):
        kv.copy_(cache)
        out[1].fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out[1].cpu().numpy(), want["scores"])
        assert np.array_equal(out[2].cpu().numpy(), want["positions"])
        assert np.array_equal(kv.double().cpu().numpy(), want["cache"])
        evict_tokens(kv.clone(), *up, 32, seen)
        torch.cuda.synchronize()


def test_no_rows():
    cache, table, lens, scores, positions = batch([10], seed=11)
    up = [torch.from_numpy(x[:0]).cuda() for x in (table, lens, scores, positions)]
    got = evict_tokens(cache.cuda(), *up, 4, up[1])
    assert got[0].shape == (0,) and got[1].shape[0] == 0
