"""Appending to a paged cache against the definition in float64: types, head dims, orders of the pairs, norms, axes, ragged
and padded batches, bad pages, advancing counts.  Every other byte of the cache stays."""

import numpy as np
import pytest
import torch

from append_cases import Tokens, check
from runtime.append import append_tokens
from runtime.rotary import rotary_frequencies

pytestmark = pytest.mark.gpu
F32, F16, BF16, FP8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


def run(batch):
    args = batch.on_gpu()
    check(batch, args, append_tokens(**args))


@pytest.mark.parametrize("dtype,kv", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, FP8), (F16, FP8), (F32, FP8)],
                         ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("dim,pairs", [(32, 16), (64, 32), (128, 64), (256, 128), (128, 32), (80, 40), (96, 24), (16, 8), (48, 0)])
@pytest.mark.parametrize("adjacent", [False, True])
def test_types_and_heads(dtype, kv, dim, pairs, adjacent):
    run(Tokens([17, 1, 64, 200], None, dim=dim, pairs=pairs, dtype=dtype, kv=kv, adjacent=adjacent, norm="shared", seed=1))
    run(Tokens([40, 9, 0, 130], [33, 1, 0, 7], dim=dim, pairs=pairs, dtype=dtype, kv=kv, adjacent=adjacent, seed=2))


@pytest.mark.parametrize("norm,weight_type,offset", [("shared", None, 0.0), ("heads", None, 1.0), ("heads", F32, 0.0),
                                                     ("shared", F32, 1.0)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=lambda t: str(t)[6:])
def test_norms(norm, weight_type, offset, dtype):
    run(Tokens([70, 5], [20, 5], dim=128, dtype=dtype, norm=norm, weight_type=weight_type, offset=offset, seed=3))
    run(Tokens([70, 5, 33], None, q_heads=3, kv_heads=3, dim=112, pairs=24, dtype=dtype, norm=norm, weight_type=weight_type,
               offset=offset, seed=4))


@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (7, 1), (28, 4), (32, 8), (64, 8), (5, 5)])
@pytest.mark.parametrize("counts", [None, [3, 1, 0, 12]])
def test_head_counts(q_heads, kv_heads, counts):
    run(Tokens([30, 17, 5, 50], counts, q_heads=q_heads, kv_heads=kv_heads, dim=128, evicting=True, seed=5))


@pytest.mark.parametrize("axes", [1, 2, 3, 4])
@pytest.mark.parametrize("counts", [None, [11, 2, 0]])
def test_axes(axes, counts):
    run(Tokens([30, 17, 5], counts, dim=128, axes=axes, seed=6, scale=0.75))
    run(Tokens([30, 17, 5], counts, dim=96, axes=axes, seed=7, adjacent=True, kv=FP8))


@pytest.mark.parametrize("block", [1, 8, 16, 24, 33])
@pytest.mark.parametrize("advance", [False, True])
@pytest.mark.parametrize("counts", [None, [9, 1, 0, 30, 2]])
def test_blocks_and_advance(block, advance, counts):
    run(Tokens([64, 23, 0 if advance else 4, 48, 31], counts, block=block, evicting=True, advance=advance, first=True, seed=8))
    run(Tokens([64, 23, 7, 48, 31], counts, block=block, advance=advance, seed=9, no_query=True))


@pytest.mark.parametrize("ahead,behind", [(0, 5), (3, 0), (2, 70)])
@pytest.mark.parametrize("advance", [False, True])
def test_tokens_of_no_row(ahead, behind, advance):
    run(Tokens([40, 3, 25], [10, 0, 25], ahead=ahead, behind=behind, evicting=True, advance=advance, seed=10))
    run(Tokens([40, 30, 25], [10, 20, 25], ahead=ahead, behind=behind, max_query=7, advance=advance, seed=11))
    run(Tokens([4, 3], [0, 0], ahead=ahead, behind=behind, advance=advance, seed=12))


@pytest.mark.parametrize("rows", [63, 64, 65, 500, 4097])
def test_many_rows(rows):
    counts = np.random.default_rng(rows).integers(0, 3, size=rows)
    counts[-1] = 0
    run(Tokens(counts + 2, counts, q_heads=2, kv_heads=1, dim=32, block=4, advance=rows % 2 == 1, behind=4, seed=13))


@pytest.mark.parametrize("rows", [1, 3, 1023, 1025, 2051, 5001])
@pytest.mark.parametrize("q_heads,kv_heads,dim", [(2, 1, 32), (20, 4, 256)])
def test_single_tokens_of_many_rows_advance(rows, q_heads, kv_heads, dim):
    """Without q_start the counts grow in the launch itself: one, two or four waves a token, one to four tokens a workgroup."""
    lens = np.random.default_rng(rows).integers(0, 9, size=rows)
    run(Tokens(lens, None, q_heads=q_heads, kv_heads=kv_heads, dim=dim, block=4, advance=True, evicting=True, seed=29))


def test_one_long_row():
    run(Tokens([3000], [2900], q_heads=4, kv_heads=2, dim=64, evicting=True, seed=14))


@pytest.mark.parametrize("advance", [False, True])
def test_pages_and_slots_that_are_not_there(advance):
    batch = Tokens([40, 33, 20, 3], [5, 4, 3, 9], evicting=True, advance=advance, seed=15, block=8)
    batch.table[0, (40 if advance else 36) // 8] = -1
    batch.table[1, (33 if advance else 30) // 8] = batch.cache.shape[0]
    batch.lens[2] = 100000  # as if it filled its pages
    batch.lens[3] = -5 if advance else 3  # fewer tokens than new ones: the first ones' slots are before the row
    run(batch)
    batch = Tokens([20, 16], [3, 4], advance=advance, seed=16, block=8, width=2, evicting=True)  # past the table's end
    run(batch)
    run(Tokens([5, 6], None, advance=advance, seed=17, width=0, evicting=True))


def test_starts_outside_the_tokens():
    batch = Tokens([30, 20, 10, 9], [8, 6, 5, 4], seed=18, evicting=True)
    batch.q_start = np.array([-4, 8, 14, 40, 50], np.int32)
    batch.max_query = 40
    run(batch)


def test_far_positions():
    """Angles of a hundred million radians, whole turns gone in float64."""
    run(Tokens([30, 20], [10, 3], dim=128, dtype=F32, evicting=True, far=2**27, seed=19))
    run(Tokens([30, 20], [10, 3], dim=128, dtype=F32, axes=3, far=2**31 - 1, seed=20))


def test_strides():
    """Heads of tensors of their own, padded rows, and a cache whose heads come before its slots."""
    batch = Tokens([40, 9, 30], [33, 1, 7], dim=64, seed=21)
    args = batch.on_gpu()
    for name in ("query", "keys", "values"):
        x = args[name]
        wide = torch.zeros(x.shape[0], x.shape[1] + 1, 2, x.shape[2] + 24, dtype=x.dtype, device="cuda")
        wide[:, 1:, 1, 8:8 + x.shape[2]] = x
        args[name] = wide[:, 1:, 1, 8:8 + x.shape[2]]
    cache = args["kv_cache"].transpose(2, 3).contiguous().transpose(2, 3)
    out = torch.zeros(batch.packed.shape[0], 3, 8, 64, dtype=BF16, device="cuda")[:, 1]
    args.update(kv_cache=cache, q_out=out)
    assert append_tokens(**args) is out
    check(batch, {**args, "kv_cache": cache.contiguous()}, out)


def test_queries_in_place():
    batch = Tokens([40, 9, 30], [33, 1, 7], dim=128, norm="shared", behind=3, seed=22)
    args = batch.on_gpu()
    assert append_tokens(**args, q_out=args["query"]) is args["query"]
    check(batch, args, args["query"])


def test_first_of_one_element():
    batch = Tokens([40, 9, 30], None, seed=23, first=True, evicting=True)
    batch.first[:] = 700
    args = batch.on_gpu()
    args["first"] = torch.full((1,), 700, dtype=torch.int32, device="cuda").expand(3)
    check(batch, args, append_tokens(**args))


def test_no_tokens():
    batch = Tokens([4, 3], [0, 0], advance=True, seed=24)
    run(batch)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("saturate", [False, True])
def test_quantised_values_are_torchs(dtype, saturate):
    """Values and scale 1: the bytes of torch's cast, clamped with saturate.  Around every border of two e4m3 values, past
    the largest, infinities and NaN."""
    codes = torch.arange(256, dtype=torch.uint8).view(FP8).float()
    finite = codes[torch.isfinite(codes)].sort().values
    border = (finite[1:] + finite[:-1]) / 2
    x = torch.cat([finite, border, border * (1 + 2.0**-20), border * (1 - 2.0**-20),
                   torch.tensor([448.0, 463.9, 464.0, 464.1, 470.0, 479.0, 480.0, 481.0, 512.0, 6e4, float("inf"), float("nan"),
                                 2.0**-10, 2.0**-11, 1e-20, 0.0])])
    x = torch.cat([x, -x]).to(dtype)
    tokens = -(-x.numel() // 32)
    x = torch.cat([x, x.new_zeros(tokens * 32 - x.numel())]).view(tokens, 1, 32).cuda()
    cache = torch.zeros(tokens, 2, 1, 1, 32, dtype=FP8, device="cuda")
    table = torch.arange(tokens, dtype=torch.int32, device="cuda").view(tokens, 1)
    append_tokens(cache, table, torch.ones(tokens, dtype=torch.int32, device="cuda"), x, x, saturate=saturate)
    wide = x.float()
    want = (wide.clamp(-448, 448) if saturate else wide).to(FP8)
    for part in (0, 1):
        got = cache[:, part, 0]
        assert torch.equal(got.float().isnan(), want.float().isnan())
        ok = ~want.float().isnan()
        assert torch.equal(got.view(torch.uint8)[ok], want.view(torch.uint8)[ok])


def test_offsets_past_32_bits():
    """Pages beyond 2^31 elements of a cache, and query rows beyond 2^31 elements of their tensor."""
    pages, block, heads, dim = 140000, 16, 8, 64
    assert pages * 2 * block * heads * dim > 2**31
    cache = torch.empty(pages, 2, block, heads, dim, dtype=BF16, device="cuda")
    batch = Tokens([19, 16], [7, 2], q_heads=8, kv_heads=heads, dim=dim, seed=25, spare=0)
    far = torch.arange(batch.cache.shape[0]) + pages - batch.cache.shape[0]
    cache[far.cuda()] = batch.cache.cuda()
    args = batch.on_gpu()
    inside = (args["table"] >= 0) & (args["table"] < batch.cache.shape[0])
    args["table"] = torch.where(inside, args["table"] + pages - batch.cache.shape[0], args["table"])
    wide = torch.empty(9, 2**28, dtype=BF16, device="cuda")
    spread = wide[:, : 8 * dim].view(9, 8, dim)
    spread.copy_(args["query"])
    out = append_tokens(**{**args, "kv_cache": cache, "query": spread}, q_out=spread)
    check(batch, {**args, "kv_cache": cache[far.cuda()]}, out)


@pytest.mark.parametrize("kv", [BF16, FP8], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("tokens", [9000, 14000, 30000])
def test_sizes_around_the_caches(kv, tokens):
    """Launches whose accesses differ by their size: the same bytes as the rows appended in pieces."""
    heads, dim, block, rows = 8, 128, 16, 3
    packed = torch.randn(tokens, 4 * heads, dim, device="cuda").to(BF16)
    query, keys, values = packed[:, :2 * heads], packed[:, 2 * heads:3 * heads], packed[:, 3 * heads:]
    counts = [tokens // 2, 1, tokens - tokens // 2 - 1]
    start = torch.tensor([0, counts[0], counts[0] + 1, tokens], dtype=torch.int32, device="cuda")
    width = -(-max(counts) // block)
    table = torch.randperm(rows * width, device="cuda").to(torch.int32).view(rows, width)
    lens = torch.tensor(counts, dtype=torch.int32, device="cuda")
    how = dict(frequencies=rotary_frequencies(dim // 2), k_scale=0.02, v_scale=0.02)
    cache = torch.zeros(rows * width, 2, block, heads, dim, dtype=kv, device="cuda")
    got = append_tokens(cache, table, lens, keys, values, q_start=start, max_query=max(counts), query=query, **how)
    want, out = torch.zeros_like(cache), torch.empty_like(got)
    for r in range(rows):
        for a in range(0, counts[r], 1000):
            b = min(counts[r], a + 1000)
            part = slice(int(start[r]) + a, int(start[r]) + b)
            out[part] = append_tokens(want, table[r:r + 1], torch.full((1,), b, dtype=torch.int32, device="cuda"), keys[part],
                                      values[part], q_start=torch.tensor([0, b - a], dtype=torch.int32, device="cuda"),
                                      max_query=b - a, query=query[part], **how)
    assert torch.equal(got, out) and torch.equal(cache.view(torch.uint8), want.view(torch.uint8))


def test_captured_steps():
    """Single tokens and prompts with advancing counts, captured once and replayed beside eager work."""
    for counts in (None, [2, 0, 1]):
        batch = Tokens([5, 9, 2], counts, evicting=True, advance=True, seed=26, width=6, kv=FP8, behind=0 if counts is None else 2)
        args, other = batch.on_gpu(), batch.on_gpu()
        n = args["keys"].shape[0]
        args["table"] = other["table"] = torch.arange(18, dtype=torch.int32, device="cuda").view(3, 6)
        pool = torch.zeros(18, 2, batch.block, 2, 64, dtype=FP8, device="cuda")
        args["kv_cache"], other["kv_cache"] = pool.clone(), pool.clone()
        start = {k: args[k].clone() for k in ("lens", "seen", "scores", "slot_positions")}
        out = torch.zeros(n, 8, 64, dtype=BF16, device="cuda")
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            append_tokens(**args, q_out=out)  # warm: what it changed is put back
        torch.cuda.synchronize()
        args["kv_cache"].copy_(pool)
        for k, v in start.items():
            args[k].copy_(v)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            append_tokens(**args, q_out=out)
        for step in range(4):
            fresh = torch.randn(n, 12, 64, device="cuda").to(BF16)
            for a in (args, other):
                a["keys"].copy_(fresh[:, :2])
                a["values"].copy_(fresh[:, 2:4])
                a["query"].copy_(fresh[:, 4:])
            graph.replay()
            want = append_tokens(**other)
            torch.cuda.synchronize()
            assert torch.equal(out, want), step
            assert torch.equal(args["kv_cache"].view(torch.uint8), other["kv_cache"].view(torch.uint8)), step
            for k in start:
                assert torch.equal(args[k], other[k]), (k, step)
        moved = 4 if counts is None else 8
        assert args["lens"].tolist() == [5 + moved, 9 + (4 if counts is None else 0), 2 + 4]


def test_two_streams():
    batches = [Tokens([700, 300, 90], [300, 2, 0], dim=128, evicting=True, seed=s) for s in (27, 28)]
    inputs, streams = [b.on_gpu() for b in batches], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for args, stream in zip(inputs, streams):
        outs.append(append_tokens(**args, stream=stream if stream is streams[0] else stream.cuda_stream))
        for size in (1 << 10, 1 << 16, 1 << 22):
            torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for batch, args, out in zip(batches, inputs, outs):
        check(batch, args, out)
