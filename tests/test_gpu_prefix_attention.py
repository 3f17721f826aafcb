"""Attention over the paged cache with shared prefixes, and the running weights, against their definition in
float64: types, head layouts, block sizes, lengths around tile, page and chunk borders, prompts and single
tokens, groups, rows that see nothing, what lies in unseen slots, strides, streams and graphs."""

import numpy as np
import pytest
import torch

from attention_cases import Batch, check
from runtime.prefix_attention import prefix_attention

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float32]


def run(batch, **more):
    args = dict(batch.on_gpu(), **more)
    out, lse = prefix_attention(**args)
    torch.cuda.synchronize()
    return out, lse, args["scores"]


@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_single_tokens(dtype, dim):
    b = Batch([1, 15, 16, 17, 63, 64, 65, 200], dim=dim, dtype=dtype, seed=dim).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("heads,group", [(1, 1), (3, 1), (1, 7), (2, 8), (1, 16), (1, 33), (5, 3)])
def test_head_layouts(heads, group):
    b = Batch([5, 130, 77], heads=heads, group=group, seed=heads * 100 + group).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("block", [1, 2, 8, 12, 16, 24, 32, 48, 64, 100])
def test_block_sizes(block):
    b = Batch([1, block, block + 1, 3 * block + 5, 150], prefixes=[2 * block + 3], block=block, seed=block).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_prompts_behind_a_prefix(dtype):
    # a row of queries alone, one with history, one token, a row of 40; 40 rows of 4 make several tiles
    b = Batch([9, 70, 33, 40], counts=[9, 21, 1, 40], prefixes=[75], dtype=dtype, seed=3).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("dim,group", [(32, 5), (64, 7), (128, 4), (256, 1)])
def test_long_prompts(dim, group):
    b = Batch([150, 301], counts=[150, 133], prefixes=[190], heads=1, group=group, dim=dim, seed=dim).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("rows", [1, 3, 70])
def test_one_prefix(rows, dtype):
    b = Batch([1 + 3 * (r % 20) for r in range(rows)], prefixes=[161], heads=1, group=4, dtype=dtype, seed=rows)
    b.with_scores()
    check(b, *run(b))


def test_groups_and_rows_of_none():
    # rows 0 and 1 and the last in no group, an empty group, an empty prefix, a group of 40 rows
    b = Batch([20 + r for r in range(50)], prefixes=[40, 55, 0, 130], borders=[2, 5, 5, 9, 49], heads=1, group=3,
              seed=8).with_scores()
    check(b, *run(b))


def test_many_groups():
    rows = 150  # more groups than a wave has lanes
    b = Batch([3 + r % 5 for r in range(rows)], prefixes=[7 + r % 11 for r in range(rows)],
              borders=list(range(rows + 1)), heads=1, group=2, dim=32, seed=9).with_scores()
    check(b, *run(b))


def test_rows_that_see_nothing():
    b = Batch([0, 5, 0, 31], seed=4).with_scores()
    check(b, *run(b))
    b = Batch([0, 5, 0], prefixes=[0, 6], borders=[0, 2, 3], seed=5).with_scores()
    check(b, *run(b))
    # more queries than own tokens: the first ones see nothing; a row of no queries
    b = Batch([3, 0, 8, 10], counts=[6, 2, 0, 4], seed=6).with_scores()
    check(b, *run(b))


def test_queries_past_the_bound_get_nothing():
    b = Batch([12, 30], counts=[12, 5], seed=7)
    b.max_query = 5
    check(b, *run(b)[:2])


@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("block", [16, 24])
def test_what_unseen_slots_hold_is_not_used(dtype, block):
    b = Batch([5, 23, 0, 40], counts=[1, 3, 1, 1], prefixes=[21], block=block, dtype=dtype, seed=11).with_scores()
    want = b.want()
    raw = b.cache.float()
    used = np.zeros(raw.shape[0:1] + raw.shape[2:3], dtype=bool)
    for pages, n in [*zip(b.table, b.lens), (b.prefix_table[0], b.prefix_lens[0])]:
        for j in range(n):
            used[pages[j // block], j % block] = True
    dirt = [np.nan] if dtype == torch.float8_e4m3fn else [np.nan, np.inf, -np.inf]
    for k, x in enumerate(dirt):
        raw.permute(0, 2, 1, 3, 4)[torch.from_numpy(~used)] = x
        b.cache = raw.to(dtype)
        out, lse, scores = run(b)
        check(b, out, lse, scores, want)


@pytest.mark.parametrize("block", [16, 24])
def test_bad_pages_are_as_if_absent(block):
    b = Batch([100, 64, 30], prefixes=[90], block=block, seed=12).with_scores()
    b.table[0, 1] = -1
    b.table[0, 3] = b.cache.shape[0]
    b.table[1, :] = 2**31 - 1  # no page at all
    b.prefix_table[0, 2] = -2**31
    check(b, *run(b))


def test_extreme_logits():
    b = Batch([300, 17], prefixes=[100], spread=400.0, seed=13).with_scores()  # one key takes all the weight
    out, lse, scores = run(b)
    want = b.want()
    assert torch.isfinite(out).all()
    gap = np.abs(lse.double().cpu().numpy() - want["lse"])
    assert np.all(gap <= 2 * (b.dim + 4) * 2.0**-24 * want["reach"] + 1e-5)
    b = Batch([300, 17], spread=0.0, seed=14).with_scores()  # equal weights
    check(b, *run(b))
    for scale in (-0.3, 0.0):
        b = Batch([90, 17], prefixes=[33], seed=15).with_scores()
        b.scale = scale
        check(b, *run(b))


def test_masked_keys_of_the_lowest_value():
    # keys that give every query the type's lowest logit: the weights stay finite and equal
    b = Batch([40], heads=1, group=4, dtype=torch.float32, seed=16)
    b.query[:] = 1.0
    b.cache[:, 0] = torch.finfo(torch.float32).min / 128
    b.scale = 1.0
    out, lse, _ = run(b)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()


def test_strides_and_layouts():
    b = Batch([33, 90, 7], counts=[2, 5, 1], prefixes=[50], heads=3, group=2, seed=17).with_scores()
    want = b.want()
    args = b.on_gpu()
    # a cache laid out [pages, heads, 2, block, dim] inside a wider buffer, padded table rows, spaced queries
    pages, _, block, heads, dim = b.cache.shape
    big = torch.full((pages, heads + 1, 2, block, dim + 16), float("nan"), dtype=b.dtype, device="cuda")
    view = big[:, :heads, :, :, :dim].permute(0, 2, 3, 1, 4)
    view.copy_(args["kv_cache"])
    table = torch.full((3, args["table"].shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    table[:, : args["table"].shape[1]] = args["table"]
    query = torch.full((b.query.shape[0], 9, dim + 8), float("nan"), dtype=b.dtype, device="cuda")
    query[:, :6, :dim] = args["query"]
    scores = torch.full((3, heads, args["scores"].shape[2] + 9), 3.0, device="cuda")
    scores[:, :, : args["scores"].shape[2]] = args["scores"]
    wide = torch.full((b.query.shape[0], 8, dim), 7.0, dtype=b.dtype, device="cuda")
    args.update(kv_cache=view, table=table[:, : args["table"].shape[1]], query=query[:, :6, :dim], scores=scores,
                out=wide[:, 1:7])
    out, lse = prefix_attention(**args)
    check(b, out, lse, scores[:, :, : b.scores.shape[2]], want)
    assert (wide[:, 0] == 7).all() and (wide[:, 7] == 7).all() and (scores[:, :, b.scores.shape[2]:] == 3).all()


def test_offsets_past_32_bits():
    # 2.7e9 elements: the pages in use are the last ones
    pages, block, heads, dim = 41000, 16, 8, 256
    cache = torch.empty(pages, 2, block, heads, dim, dtype=torch.bfloat16, device="cuda")
    b = Batch([40, 21], prefixes=[37], heads=heads, group=2, dim=dim, seed=18).with_scores()
    n = b.cache.shape[0]
    cache[pages - n:] = b.cache.cuda()
    args = b.on_gpu()
    live = torch.from_numpy(b.table < n).cuda()
    args["table"] = torch.where(live, args["table"] + (pages - n), args["table"])
    args["prefix_table"] = args["prefix_table"] + (pages - n)
    out, lse = prefix_attention(**dict(args, kv_cache=cache))
    check(b, out, lse, args["scores"])


def test_a_long_row_over_many_chunks():
    b = Batch([5000, 1], heads=1, group=2, dim=32, seed=19).with_scores()
    check(b, *run(b))


def test_equal_calls_give_equal_bits():
    b = Batch([300, 5, 2000], counts=[4, 4, 30], prefixes=[700], heads=2, group=3, seed=20).with_scores()
    first = run(b)
    for _ in range(3):
        again = run(b)
        assert all(torch.equal(x, y) for x, y in zip(first, again))


def test_another_stream():
    b = Batch([300, 5, 90], prefixes=[70], seed=21).with_scores()
    args = b.on_gpu()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out, lse = prefix_attention(**args)
    stream.synchronize()
    check(b, out, lse, args["scores"])
    args = b.on_gpu()
    torch.cuda.synchronize()
    out, lse = prefix_attention(**args, stream=stream)
    stream.synchronize()
    check(b, out, lse, args["scores"])


def test_graph_replays():
    b = Batch([300, 5, 90, 41], counts=[1, 4, 20, 1], prefixes=[170], seed=22).with_scores()
    args = b.on_gpu()
    start = args["scores"].clone()
    out, lse = torch.empty_like(args["query"]), torch.empty(26, 8, device="cuda")
    want_out, want_lse = prefix_attention(**args)
    want_scores = args["scores"].clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            prefix_attention(**args, out=out, lse=lse)
    for _ in range(4):
        args["scores"].copy_(start)
        out.zero_()
        lse.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want_out) and torch.equal(lse, want_lse) and torch.equal(args["scores"], want_scores)
        prefix_attention(**b.on_gpu())  # other work of the program between the replays
        torch.cuda.synchronize()


def test_no_rows():
    b = Batch([4], seed=23)
    args = b.on_gpu()
    args.update(query=args["query"][:0], table=args["table"][:0], lens=args["lens"][:0])
    out, lse = prefix_attention(**args)
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)


def test_scores_decay_without_queries():
    b = Batch([20, 5], counts=[0, 0], seed=24).with_scores(decay=0.5)
    out, lse, scores = run(b)
    assert out.shape[0] == 0
    want = b.want()["scores"]
    assert np.abs(scores.cpu().numpy() - want).max() <= np.abs(want).max() * 2.0**-24
