"""The budgeted cache on the GPU: its appends against the host's, bit for bit, and with a rotation its whole loop (a shared
prefix, ragged padded prompts, decode steps, evictions) against the definitions over the cache as it stands."""

import numpy as np
import pytest
import torch

from append_cases import bound
from attention_cases import bounds
from oracle import append as oracle
from oracle import attention
from runtime.budgeted_cache import BudgetedCache
from runtime.rotary import rotary_frequencies, section_axes
from test_gpu_budgeted_cache import check_trim

ROWS, HEADS = 3, 2
F32, F16, BF16, FP8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


def same(here, host):
    for name in ("kv", "lens", "seen", "positions", "scores"):
        a, b = getattr(here, name).cpu(), getattr(host, name)
        if name == "kv":
            a, b = a[1:].view(torch.uint8), b[1:].view(torch.uint8)  # page 0 is nobody's
        assert torch.equal(a, b), name
    assert here.longest == host.longest


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16, FP8], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("dim", [32, 48, 40, 256, 272])  # 40 and 272 have no kernel
@pytest.mark.parametrize("given", [F32, F16, BF16, torch.float64], ids=lambda t: str(t)[6:])
def test_appends_are_the_hosts(dtype, dim, given):
    gen = torch.Generator().manual_seed(dim)
    caches = [BudgetedCache(ROWS, HEADS, dim, budget=24, slack=16, prefix=5, block=4, dtype=dtype, device=d) for d in ("cuda", "cpu")]

    def both(call):
        for c in caches:
            call(c, c.kv.device)

    def tokens(n, spread=1.0):
        rows = (spread * torch.randn(n, 2 * HEADS, dim, generator=gen)).to(given)
        if given == F32:
            rows[0, 0, :5] = torch.tensor([1e-39, -1e-42, 3e38, -0.0, float("inf")])
        return rows

    def step(rows, q_start=None, longest=1):
        both(lambda c, d: c.append(rows[:, :HEADS].to(d), rows[:, HEADS:].to(d), None if q_start is None else q_start.to(d), longest))
        same(*caches)

    prefix = tokens(5)
    both(lambda c, d: c.set_prefix(prefix[:, :HEADS].to(d), prefix[:, HEADS:].to(d)))
    same(*caches)
    for c in caches:
        c.scores.fill_(3.0)
    step(tokens(17), torch.tensor([2, 9, 9, 14], dtype=torch.int64), 6)  # padding on both sides, a row past max_query
    step(tokens(ROWS, 200.0))
    step(tokens(9), torch.tensor([0, 1, 5, 9], dtype=torch.int32), 4)
    wide = tokens(ROWS)
    caches[0].append(*(torch.stack([x, x], -1)[..., 0].cuda() for x in (wide[:, :HEADS], wide[:, HEADS:])))  # elements apart
    caches[1].append(wide[:, :HEADS], wide[:, HEADS:])
    same(*caches)
    odd = torch.zeros(ROWS, HEADS, dim + 1, dtype=given)
    odd[..., 1:] = tokens(ROWS)[:, :HEADS]
    both(lambda c, d: c.append(odd.to(d)[..., 1:], odd.to(d)[..., 1:].to(F16)))  # off 16 bytes, types of their own
    same(*caches)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16], ids=lambda t: str(t)[6:])
def test_every_16_bit_value_is_kept(dtype):
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    x = bits.view(dtype).view(32, 1, 2048)[..., :2048].reshape(256, 1, 256).cuda()
    cache = BudgetedCache(256, 1, 256, budget=1, slack=1, block=1, dtype=dtype)
    cache.append(x, x)
    got = cache.kv[cache.table[:, 0].long(), :, 0]  # [rows, 2, 1, 256]
    for part in (0, 1):
        a, b = got[:, part], x
        assert torch.equal(a.isnan(), b.isnan())
        assert torch.equal(a.view(torch.int16)[~b.isnan()], b.view(torch.int16)[~b.isnan()])


def check_attend(cache, query, scale, q_start=None, longest=1):
    """The attention over the cache as it stands; tokens of no row get 0 and -inf."""
    shared = cache.prefix_table is not None
    want = attention.attend(
        query.double().cpu().numpy(), cache.kv.double().cpu().numpy(), cache.table.cpu().numpy(), cache.lens.cpu().numpy(),
        scale, None if q_start is None else q_start.cpu().numpy(), longest,
        cache.prefix_table.cpu().numpy() if shared else None, cache.prefix_len.cpu().numpy() if shared else None, None,
        cache.k_scale, cache.v_scale, cache.scores.cpu().numpy(), cache.decay)
    out, lse = (x.double().cpu().numpy() for x in cache.attend(query, scale, q_start, longest))
    out_bound, lse_bound, relative = bounds(want, query.shape[2], query.dtype)
    dead = np.isneginf(want["lse"])
    assert np.array_equal(np.isneginf(lse), dead) and np.all(out[dead] == 0)
    assert np.all(np.abs(out - want["out"]) <= out_bound)
    assert np.all(np.abs(np.where(dead, 0, lse) - np.where(dead, 0, want["lse"])) <= lse_bound)
    off = np.abs(cache.scores.double().cpu().numpy() - want["scores"])
    group = query.shape[1] // cache.kv.shape[3]
    assert np.all(off <= (2 * relative.max() + (longest * group + 8) * 2.0**-24) * np.abs(want["scores"]) + 2.0**-100)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32, FP8], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("prefix,axes", [(0, 0), (37, 0), (21, 3)])
def test_the_loop_with_a_rotation(dtype, prefix, axes):
    rows, group, dim, pairs = 5, 3, 64, 24
    fp8 = dtype == FP8
    kind = BF16 if fp8 else dtype
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    weights = [(1 + 0.2 * torch.randn(n, dim, generator=gen, device="cuda")).to(kind) for n in (HEADS * group, HEADS)]
    frequencies = rotary_frequencies(pairs)
    rotation = dict(frequencies=frequencies, q_weight=weights[0], k_weight=weights[1], rotary_scale=0.9)
    if axes:
        rotation["axes"] = section_axes(8, 8, 8, interleaved=True)
    cache = BudgetedCache(rows, HEADS, dim, budget=40, slack=24, prefix=prefix, block=16, dtype=dtype, recent=8, sinks=2,
                          decay=0.75, k_scale=0.02 if fp8 else 1.0, v_scale=0.02 if fp8 else 1.0, rotation=rotation)
    turn = dict(frequencies=frequencies.cpu().numpy(), axes=None if not axes else rotation["axes"].cpu().numpy(), rotary_scale=0.9,
                q_weight=weights[0].double().cpu().numpy(), k_weight=weights[1].double().cpu().numpy(), k_scale=cache.k_scale,
                v_scale=cache.v_scale)

    def projected(n):
        x = torch.randn(n, HEADS * (group + 2), dim, generator=gen, device="cuda").to(kind)
        return x[:, :HEADS * group], x[:, HEADS * group:HEADS * (group + 1)], x[:, HEADS * (group + 1):]

    def positions_of(n):
        return torch.randint(0, 4000, (axes, n), generator=gen, device="cuda", dtype=torch.int32) if axes else None

    def check(want, query, angle):
        wrote, got = want["wrote"], cache.kv.double().cpu().numpy()
        assert np.array_equal(got[~wrote], want["cache"][~wrote])
        assert np.all(np.abs(got - want["cache"]) <= bound(want["cache"], want["reach"], dtype, dim, True, angle))
        if query is not None:
            limit = bound(want["query"], want["query_reach"], kind, dim, True, angle, False)
            assert np.all(np.abs(query.double().cpu().numpy() - want["query"]) <= limit)
            for name in ("lens", "seen", "scores", "slot_positions"):
                mine = cache.positions if name == "slot_positions" else getattr(cache, name)
                assert np.array_equal(mine.cpu().numpy(), want[name]), name

    def append(n, q_start=None, longest=1):
        query, keys, values = projected(n)
        where = positions_of(n)
        host = [x.double().cpu().numpy() for x in (keys, values, query)]
        want = oracle.append(
            cache.kv.double().cpu().numpy(), cache.table.cpu().numpy(), cache.lens.cpu().numpy(), host[0], host[1],
            None if q_start is None else q_start.cpu().numpy(), longest, host[2], None if where is None else where.cpu().numpy(),
            seen=cache.seen.cpu().numpy(), first=np.full(rows, prefix), scores=cache.scores.cpu().numpy(),
            slot_positions=cache.positions.cpu().numpy(), advance=True, **turn)
        out = cache.append(keys, values, q_start, longest, query=query, positions=where)
        check(want, out, 4000.0)
        return out

    scale = dim**-0.5
    if prefix:
        _, keys, values = projected(prefix)
        where = positions_of(prefix)
        host = [x.double().cpu().numpy() for x in (keys, values)]
        want = oracle.append(cache.kv.double().cpu().numpy(), cache.prefix_table.cpu().numpy(), np.array([prefix]), *host,
                             np.array([0, prefix]), prefix, positions=None if where is None else where.cpu().numpy(), **turn)
        cache.set_prefix(keys, values, where)
        check(want, None, 4000.0)
    start = torch.tensor([3, 33, 33, 67, 68, 110], dtype=torch.int32, device="cuda")  # padded on both sides
    check_attend(cache, append(120, start, 42), scale, start, 42)
    trims = 0
    for _ in range(30):
        check_attend(cache, append(rows), scale)
        if cache.full:
            check_trim(cache)
            trims += 1
    assert trims >= 1


def test_refusals():
    rows = torch.zeros(2, HEADS, 32)
    plain = BudgetedCache(2, HEADS, 32, budget=4, prefix=3, device="cpu")
    with pytest.raises(ValueError, match="rotation"):
        plain.append(rows, rows, query=rows)
    with pytest.raises(ValueError, match="rotation"):
        plain.append(rows, rows, positions=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="rotation"):
        plain.set_prefix(rows, rows, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="base"):
        BudgetedCache(2, HEADS, 32, budget=4, rotation=dict(base=10000.0), device="cpu")
    cache = BudgetedCache(2, HEADS, 32, budget=4, rotation=dict(frequencies=rotary_frequencies(16, device="cpu")), device="cpu")
    with pytest.raises(ValueError, match="device tensor"):
        cache.append(rows.bfloat16(), rows.bfloat16())
    assert cache.longest == 0


def test_a_refused_prefix_leaves_none():
    cache = BudgetedCache(2, HEADS, 32, budget=4, prefix=3, rotation=dict(frequencies=rotary_frequencies(16, device="cpu")), device="cpu")
    rows = torch.zeros(3, HEADS, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device tensor"):
        cache.set_prefix(rows, rows)
    assert cache.prefix_len.item() == 0
