"""Norms and rotations of query and key heads without a cache, against the definition in float64."""

import numpy as np
import pytest
import torch

from append_cases import bound
from oracle import append as oracle
from runtime.rotary import rotary_frequencies, rotate_heads, section_axes

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def case(tokens, q_heads, kv_heads, dim, pairs, dtype, seed, far=100000, axes=0, adjacent=False, norm=None, weight_type=None,
         offset=0.0, scale=1.0, eps=1e-6, spread=1.0):
    """(arguments of rotate_heads on the GPU, a function that checks its result)."""
    rng = np.random.default_rng(seed)
    packed = torch.from_numpy(spread * rng.standard_normal((tokens, q_heads + kv_heads, dim))).float().to(dtype)
    positions = rng.integers(0, far, size=(max(1, axes), tokens)).astype(np.int32)
    frequencies = 10000.0 ** -(np.arange(pairs) / max(1, pairs)) if pairs else None
    axis = rng.integers(0, axes, size=pairs).astype(np.int32) if axes else None
    weights = [None, None]
    if norm:
        shapes = ((q_heads, dim), (kv_heads, dim)) if norm == "heads" else ((dim,), (dim,))
        weights = [torch.from_numpy(1 - offset + 0.3 * rng.standard_normal(s)).float().to(weight_type or dtype) for s in shapes]
    up = packed.cuda()
    args = dict(query=up[:, :q_heads], key=up[:, q_heads:] if kv_heads else None,
                positions=torch.from_numpy(positions if axes else positions[0]).cuda() if pairs else None,
                frequencies=torch.from_numpy(frequencies).cuda() if pairs else None,
                axes=None if axis is None else torch.from_numpy(axis).cuda(), adjacent=adjacent, rotary_scale=scale,
                q_weight=None if weights[0] is None else weights[0].cuda(),
                k_weight=None if weights[1] is None or not kv_heads else weights[1].cuda(), eps=eps, weight_offset=offset)

    def check(query, key):
        for got, heads, w in ((query, packed[:, :q_heads], weights[0]), (key, packed[:, q_heads:], weights[1])):
            if not kv_heads and got is None:
                continue
            x = heads.double().numpy()
            want, reach = np.zeros(x.shape), np.zeros(x.shape)
            for t in range(tokens):
                want[t], reach[t] = oracle.rotate(x[t], None if w is None else w.double().numpy(), eps, offset, positions[:, t],
                                                  frequencies, axis, adjacent, scale)
            off = np.abs(got.double().cpu().numpy() - want)
            assert np.all(off <= bound(want, reach, dtype, dim, norm is not None, float(far) if pairs else 0.0, False)), off.max()

    return args, check


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("dim,pairs", [(16, 8), (32, 16), (48, 16), (64, 16), (64, 32), (80, 40), (112, 56), (128, 64), (128, 0),
                                       (192, 32), (256, 128), (256, 64), (240, 120)])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("norm", [None, "shared", "heads"])
def test_shapes(dtype, dim, pairs, adjacent, norm):
    args, check = case(5, 6, 2, dim, pairs, dtype, 1, adjacent=adjacent, norm=norm)
    check(*rotate_heads(**args))


@pytest.mark.parametrize("tokens", [1, 2, 3, 129, 1100, 2500])
@pytest.mark.parametrize("q_heads,kv_heads", [(1, 0), (1, 1), (9, 3), (32, 8)])
def test_sizes(tokens, q_heads, kv_heads):
    args, check = case(tokens, q_heads, kv_heads, 32, 16, BF16, 2, norm="shared", weight_type=F32, offset=1.0)
    check(*rotate_heads(**args))


@pytest.mark.parametrize("axes", [1, 2, 3, 5])
@pytest.mark.parametrize("dtype", [F32, F16], ids=lambda t: str(t)[6:])
def test_axes(axes, dtype):
    args, check = case(70, 4, 4, 80, 40, dtype, 3, axes=axes, scale=1.3)
    check(*rotate_heads(**args))


def test_an_axis_that_is_not_there_is_position_0():
    args, _ = case(9, 2, 1, 32, 16, F32, 4, axes=2)
    args["axes"][3], args["axes"][5] = -1, 2
    query, _ = rotate_heads(**args)
    for p in (3, 5):
        assert torch.equal(query[..., p], args["query"][..., p]) and torch.equal(query[..., 16 + p], args["query"][..., 16 + p])


@pytest.mark.parametrize("far", [2**24 + 3, 2**31 - 1])
def test_far_positions(far):
    args, check = case(40, 2, 2, 128, 64, F32, 5, far=far)
    check(*rotate_heads(**args))


def test_negative_positions_turn_back():
    args, _ = case(33, 4, 2, 64, 32, F32, 6, norm=None)
    query, key = rotate_heads(**args)
    back, key_back = rotate_heads(query, key, -args["positions"], args["frequencies"])
    # two rotations, each off by what `bound` counts of the sum of a pair's magnitudes
    for got, x in ((back, args["query"]), (key_back, args["key"])):
        reach = x.abs().double().view(33, -1, 2, 32).sum(2, keepdim=True).expand(-1, -1, 2, -1).reshape(x.shape).cpu().numpy()
        limit = 2 * bound(x.double().cpu().numpy(), 1.5 * reach, F32, 64, False, 1e5, False)
        assert np.all(np.abs((got - x).double().cpu().numpy()) <= limit)


def test_in_place_and_given_outputs():
    args, check = case(300, 8, 2, 128, 64, BF16, 7, norm="shared")
    out, k_out = torch.zeros(300, 2, 8, 128, dtype=BF16, device="cuda")[:, 1], torch.zeros(300, 2, 128, dtype=BF16, device="cuda")
    got = rotate_heads(**args, q_out=out, k_out=k_out)
    assert got[0] is out and got[1] is k_out
    check(out, k_out)
    got = rotate_heads(**args, q_out=args["query"], k_out=args["key"])
    assert got[0] is args["query"] and got[1] is args["key"]
    check(*got)


def test_one_head_and_one_token_of_any_stride():
    rows = torch.randn(3, 100, device="cuda", dtype=F32)  # rows of 400 bytes
    one = rows[0:1, 4:36].unsqueeze(1)
    at = torch.full((1,), 7, dtype=torch.int32, device="cuda")
    got, _ = rotate_heads(one, None, at, rotary_frequencies(16))
    want, _ = rotate_heads(one.clone(), None, at, rotary_frequencies(16))
    assert torch.equal(got, want)
    with pytest.raises(ValueError, match="16 bytes"):
        rotate_heads(rows[0:1, 1:33].unsqueeze(1), None, at, rotary_frequencies(16))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: str(t)[6:])
def test_norms_of_extremes(dtype):
    """Squares past float32, all zeros, infinities and NaN: as the definition has them, head by head."""
    x = torch.randn(7, 1, 64, device="cuda").to(dtype)
    x[0] *= 1e30
    x[1] *= 2.0**126
    x[2] = 0
    x[3, 0, 5] = float("inf")
    x[4, 0, 7] = float("nan")
    x[5] *= 1e-25
    w = torch.ones(64, dtype=dtype, device="cuda")
    got, _ = rotate_heads(x, None, None, None, q_weight=w)
    wide = x.double()
    want = wide / torch.sqrt((wide * wide).mean(-1, keepdim=True) + 1e-6)
    assert torch.all(got[2] == 0)
    assert torch.all(got[3, 0, torch.arange(64, device="cuda") != 5] == 0) and torch.isnan(got[3, 0, 5])
    assert torch.all(torch.isnan(got[4]))
    for t in (0, 1, 5, 6):
        a, b = got[t].double().cpu().numpy(), want[t].cpu().numpy()
        assert np.all(np.abs(a - b) <= bound(b, np.abs(b), dtype, 64, True, 0.0, False)), t


def test_a_pair_that_does_not_turn_meets_nothing():
    """Elements behind the rotated ones do not mix: an infinity there stays alone."""
    x = torch.randn(2, 1, 64, device="cuda")
    x[:, :, 40] = float("inf")
    at = torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    got, _ = rotate_heads(x, None, at, rotary_frequencies(16))
    rest = torch.arange(64, device="cuda") >= 32
    assert torch.equal(got[..., rest], x[..., rest]) and torch.all(torch.isfinite(got[..., ~rest]))


def test_captured():
    args, _ = case(77, 8, 2, 128, 64, BF16, 8, norm="shared")
    out, k_out = torch.zeros(77, 8, 128, dtype=BF16, device="cuda"), torch.zeros(77, 2, 128, dtype=BF16, device="cuda")
    rotate_heads(**args, q_out=out, k_out=k_out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rotate_heads(**args, q_out=out, k_out=k_out)
    for _ in range(3):
        args["query"].copy_(torch.randn(77, 8, 128, device="cuda"))
        args["positions"].add_(11)
        graph.replay()
        query, key = rotate_heads(**args)
        torch.cuda.synchronize()
        assert torch.equal(out, query) and torch.equal(k_out, key)


def test_sections_on_the_device():
    axes = section_axes(8, 12, 12)
    assert axes.is_cuda and axes.tolist() == [0] * 8 + [1] * 12 + [2] * 12
    n = torch.arange(6, dtype=torch.int32, device="cuda")
    x = torch.randn(6, 2, 64, device="cuda")
    same, _ = rotate_heads(x, None, n.expand(3, 6).contiguous(), rotary_frequencies(32), axes=axes)
    want, _ = rotate_heads(x, None, n, rotary_frequencies(32))
    assert torch.equal(same, want)  # text: every axis the same position


@pytest.mark.parametrize("tokens,dim", [(2**25 + 3, 16), (2**24 + 5, 128)])
def test_more_waves_than_a_launch_has_threads_for(tokens, dim):
    """A token a wave where two or four would pass 2^32 threads: slices of the call's result are those of calls of their own."""
    x = torch.empty(tokens, 1, dim, dtype=BF16, device="cuda")
    for a in range(0, tokens, 2**22):
        x[a:a + 2**22] = torch.randn(min(2**22, tokens - a), 1, dim, device="cuda")
    at = torch.arange(tokens, dtype=torch.int32, device="cuda")
    f = rotary_frequencies(dim // 2)
    got, _ = rotate_heads(x, None, at, f)
    for a in (0, 2**22 - 9, 2**24 - 17, tokens - 1000):
        part = slice(a, a + 1000)
        want, _ = rotate_heads(x[part], None, at[part], f)
        assert torch.equal(got[part], want)


@pytest.mark.parametrize("pairs,dim,dtype", [(64, 128, BF16), (40, 80, F16), (64, 128, F32), (32, 128, BF16)])
@pytest.mark.parametrize("tokens", [9000, 21000, 60000])
def test_sizes_around_the_caches(pairs, dim, dtype, tokens):
    """Launches of 60 MB to 2 GB, whose accesses differ: slices of the result are those of small calls."""
    x = torch.randn(tokens, 16, dim, device="cuda").to(dtype)
    at = torch.arange(tokens, dtype=torch.int32, device="cuda") + 1000
    f, w = rotary_frequencies(pairs), torch.rand(dim, device="cuda").to(dtype)
    for weight in (None, w):
        query, key = rotate_heads(x[:, :12], x[:, 12:], at, f, q_weight=weight, k_weight=weight)
        for a in (0, tokens // 2 + 1, tokens - 700):
            part = slice(a, a + 700)
            want = rotate_heads(x[part, :12], x[part, 12:], at[part], f, q_weight=weight, k_weight=weight)
            assert torch.equal(query[part], want[0]) and torch.equal(key[part], want[1])


@pytest.mark.parametrize("q_heads,kv_heads,dim,pairs", [(1, 1, 96, 48), (3, 1, 128, 32), (2, 1, 64, 32), (1, 1, 256, 128), (5, 2, 32, 16),
                                                        (1, 0, 80, 40), (4, 1, 128, 0), (1, 1, 16, 8), (3, 1, 240, 120)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("norm", [None, "shared", "heads"])
def test_few_heads_of_many_tokens(q_heads, kv_heads, dim, pairs, dtype, norm):
    """Where a token's heads are few a wave takes several tokens: the same bits as small calls, which take them one by one."""
    tokens = 8 * 1024 + 13
    for axes, adjacent in ((0, False), (3, True)):
        args, check = case(tokens, q_heads, kv_heads, dim, pairs, dtype, 9, axes=axes if pairs else 0, adjacent=adjacent, norm=norm)
        query, key = rotate_heads(**args)
        for a in range(0, tokens, 2000):
            part = slice(a, a + 2000)
            where = {} if not pairs else {"positions": args["positions"][..., part].contiguous()}
            want = rotate_heads(**{**args, **where, "query": args["query"][part], "key": None if key is None else args["key"][part]})
            assert torch.equal(query[part], want[0]) and (key is None or torch.equal(key[part], want[1]))
        got = rotate_heads(**args, q_out=args["query"], k_out=args["key"])
        assert torch.equal(got[0], query) and (key is None or torch.equal(got[1], key))


@pytest.mark.parametrize("dtype,norm", [(F32, "heads"), (F16, "shared"), (BF16, None)])
def test_few_heads_against_the_definition(dtype, norm):
    args, check = case(8 * 1024 + 3, 1, 1, 32, 16, dtype, 10, axes=2, norm=norm)
    check(*rotate_heads(**args))


def test_axes_of_one_row_of_positions():
    """Positions that are one row seen as three."""
    n = torch.arange(50, dtype=torch.int32, device="cuda")
    x = torch.randn(50, 2, 64, device="cuda")
    got, _ = rotate_heads(x, None, n.expand(3, 50), rotary_frequencies(32), axes=section_axes(8, 12, 12))
    want, _ = rotate_heads(x, None, n, rotary_frequencies(32))
    assert torch.equal(got, want)


def test_no_tokens():
    x = torch.empty(0, 4, 64, device="cuda", dtype=BF16)
    query, key = rotate_heads(x, x, torch.empty(0, dtype=torch.int32, device="cuda"), rotary_frequencies(32))
    assert query.shape == key.shape == (0, 4, 64)
