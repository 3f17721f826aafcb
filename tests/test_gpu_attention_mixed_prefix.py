"""Rows of a few queries each (more than a narrow tile holds, fewer than a wide one) and prompts among single tokens behind
shared prefixes: the prefixes read once for their groups, the own keys by row, joined; against the definition in float64."""

import numpy as np
import pytest
import torch

from attention_cases import Batch, check
from runtime.prefix_attention import prefix_attention

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float8_e4m3fn]
LONG = 1 << 20  # tokens that a prefix may have: enough to read it together


def long_prefixes(b):
    """The batch with a prefix table wide enough for LONG tokens; what is past a prefix is no page."""
    table = np.full((len(b.prefix_table), LONG // b.block), -7, np.int32)
    table[:, : b.prefix_table.shape[1]] = b.prefix_table
    b.prefix_table = table
    return b


def run(batch, **more):
    args = dict(batch.on_gpu(), **more)
    out, lse = prefix_attention(**args)
    torch.cuda.synchronize()
    return out, lse, args["scores"]


@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_drafts_behind_a_prefix(dtype, dim):
    b = long_prefixes(Batch([5, 17, 64, 90, 6, 33], counts=[5, 17, 16, 9, 6, 1], prefixes=[137], heads=2, group=4, dim=dim,
                            dtype=dtype, seed=dim)).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_a_prompt_among_single_tokens(dtype):
    b = long_prefixes(Batch([1 + 5 * (r % 9) for r in range(12)] + [290] + [20] * 13, counts=[1] * 12 + [270] + [1] * 13,
                            prefixes=[150], heads=1, group=2, dtype=dtype, seed=3)).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("heads,group,queries", [(1, 16, 2), (3, 5, 7), (2, 1, 20), (1, 32, 1), (1, 8, 40)])
def test_head_layouts(heads, group, queries):
    b = long_prefixes(Batch([queries + 3 * r for r in range(9)], counts=[queries] * 9, prefixes=[70, 40], borders=[0, 6, 9],
                            heads=heads, group=group, seed=heads * 100 + group)).with_scores()
    check(b, *run(b))


def test_groups_of_every_kind():
    # a row ahead of the groups, an empty group, one of no tokens, one row alone, rows behind all groups
    lens, counts = [9, 30, 12, 0, 25, 40, 19, 30, 8], [9, 9, 7, 9, 5, 9, 1, 0, 8]
    b = long_prefixes(Batch(lens, counts=counts, prefixes=[50, 90, 0, 33], borders=[1, 3, 3, 5, 7], heads=2, group=3,
                            seed=8)).with_scores()
    check(b, *run(b))


def test_own_keys_of_several_chunks():
    b = long_prefixes(Batch([1600, 700, 30], counts=[20, 18, 19], prefixes=[700], heads=1, group=1, dim=32, seed=5)).with_scores()
    check(b, *run(b))


def test_prefixes_of_many_tiles_and_pieces():
    b = long_prefixes(Batch([9 + r % 7 for r in range(70)], counts=[9] * 70, prefixes=[1700, 530], borders=[0, 40, 70],
                            heads=1, group=2, dim=32, seed=6))
    check(b, *run(b))


def test_rows_that_see_only_their_prefix_or_nothing():
    b = long_prefixes(Batch([3, 0, 5, 40], counts=[20, 18, 0, 20], prefixes=[0, 40], borders=[0, 2, 3], heads=1, group=2,
                            seed=14)).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("block", [1, 12, 16, 24, 100])
def test_block_sizes_and_bad_pages(block):
    b = long_prefixes(Batch([170, 131, 90], counts=[20, 18, 17], prefixes=[130], heads=1, group=2, block=block,
                            seed=block)).with_scores()
    b.table[0, 1] = -1
    b.table[2, :] = 2**31 - 1
    b.prefix_table[0, 0] = b.cache.shape[0]
    check(b, *run(b))


def test_tokens_of_no_row():
    b = long_prefixes(Batch([100, 20, 80], counts=[30, 10, 10], prefixes=[60], heads=2, group=2, dim=32, seed=15))
    want = b.want()
    b.max_query = 17
    bounded = b.want()
    args = b.on_gpu()
    query = torch.randn(3 + 50 + 2, 4, 32, dtype=torch.bfloat16, device="cuda")
    query[3:53] = args["query"]
    args.update(query=query, q_start=args["q_start"] + 3)
    for most, held in ((17, bounded), (30, want)):
        out, lse = torch.full_like(query, 9.0), torch.full((55, 4), 9.0, device="cuda")
        prefix_attention(**{**args, "max_query": most}, out=out, lse=lse)
        for part in (slice(0, 3), slice(53, 55)):
            assert not out[part].any() and torch.isneginf(lse[part]).all()
        check(b, out[3:53], lse[3:53], None, held)


def test_graph_replays_and_equal_bits():
    b = long_prefixes(Batch([300, 25, 90, 41], counts=[20, 9, 20, 1], prefixes=[170], seed=22)).with_scores()
    args = b.on_gpu()
    start = args["scores"].clone()
    out, lse = torch.empty_like(args["query"]), torch.empty(50, 8, device="cuda")
    want_out, want_lse = prefix_attention(**args)
    want_scores = args["scores"].clone()
    check(b, want_out, want_lse, want_scores)
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
        prefix_attention(**b.on_gpu())
        torch.cuda.synchronize()
