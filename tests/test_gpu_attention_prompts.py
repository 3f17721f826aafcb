"""Attention of many query rows at once (prompt chunks over their prefix and their own keys, a group's queries over its
prefix) against its definition in float64: types, head dims, ragged tiles, chunks of keys, masks, unseen slots."""

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
def test_chunks_with_history_and_prefix(dtype, dim):
    b = Batch([210, 75, 33], counts=[140, 75, 2], prefixes=[137], heads=1, group=2, dim=dim, dtype=dtype,
              seed=dim).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_single_tokens_of_a_large_group(dtype, dim):
    b = Batch([1 + 5 * (r % 9) for r in range(45)], prefixes=[150], heads=2, group=3, dim=dim, dtype=dtype, seed=dim + 1)
    check(b, *run(b))


@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_keys_of_several_chunks(dtype):
    # 2300 keys on one axis: 700 of the prefix, then the row's own; the second row's end inside the prefix's chunks
    b = Batch([1600, 70], counts=[70, 66], prefixes=[700], heads=1, group=1, dim=32, dtype=dtype, seed=5).with_scores()
    check(b, *run(b))


def test_a_long_prefix_in_several_chunks():
    b = Batch([3 + r % 7 for r in range(70)], prefixes=[1700, 530], borders=[0, 40, 70], heads=1, group=2, dim=32, seed=6)
    check(b, *run(b))


@pytest.mark.parametrize("heads,group", [(1, 64), (3, 5), (2, 16), (1, 1)])
def test_head_layouts(heads, group):
    b = Batch([90, 70], counts=[70, 66], prefixes=[40], heads=heads, group=group, seed=heads * 100 + group).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("block", [1, 2, 8, 12, 24, 32, 48, 100])
def test_block_sizes(block):
    b = Batch([70, 131], counts=[70, 80], prefixes=[2 * block + 3], heads=1, group=2, block=block, seed=block).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("block", [16, 24])
def test_what_unseen_slots_hold_is_not_used(dtype, block):
    b = Batch([75, 100], counts=[75, 66], prefixes=[21], heads=1, group=2, block=block, dtype=dtype, seed=11).with_scores()
    want = b.want()
    raw = b.cache.float()
    used = np.zeros(raw.shape[0:1] + raw.shape[2:3], dtype=bool)
    for pages, n in [*zip(b.table, b.lens), (b.prefix_table[0], b.prefix_lens[0])]:
        for j in range(n):
            used[pages[j // block], j % block] = True
    dirt = [np.nan] if dtype == torch.float8_e4m3fn else [np.nan, np.inf, -np.inf]
    for x in dirt:
        raw.permute(0, 2, 1, 3, 4)[torch.from_numpy(~used)] = x
        b.cache = raw.to(dtype)
        check(b, *run(b), want)


@pytest.mark.parametrize("block", [16, 24])
def test_bad_pages_are_as_if_absent(block):
    b = Batch([100, 70, 90], counts=[70, 64, 66], prefixes=[90], heads=1, group=2, block=block, seed=12).with_scores()
    b.table[0, 1] = -1
    b.table[0, 3] = b.cache.shape[0]
    b.table[1, :] = 2**31 - 1  # no page at all
    b.prefix_table[0, 2] = -2**31
    check(b, *run(b))


def test_rows_that_see_nothing():
    # more queries than tokens, no tokens at all, no queries
    b = Batch([30, 0, 5, 90], counts=[70, 66, 0, 90], heads=1, group=2, seed=13).with_scores()
    check(b, *run(b))
    b = Batch([30, 0, 5, 90], counts=[70, 66, 0, 90], prefixes=[0, 40], borders=[0, 2, 3], heads=1, group=2, seed=14)
    check(b, *run(b))


@pytest.mark.parametrize("keys", [100, 1500])
def test_tokens_of_no_row_get_nothing(keys):
    b = Batch([keys, 80], counts=[90, 70], heads=2, group=2, dim=32, seed=15)
    want = b.want()
    b.max_query = 66  # the last 24 tokens of the first row and 4 of the second are past it
    bounded = b.want()
    args = b.on_gpu()
    query = torch.randn(3 + 160 + 2, 4, 32, dtype=torch.bfloat16, device="cuda")
    query[3:163] = args["query"]
    args.update(query=query, q_start=args["q_start"] + 3)
    out, lse = torch.full_like(query, 9.0), torch.full((165, 4), 9.0, device="cuda")
    prefix_attention(**args, out=out, lse=lse)
    for part in (slice(0, 3), slice(163, 165)):
        assert not out[part].any() and torch.isneginf(lse[part]).all()
    check(b, out[3:163], lse[3:163], None, bounded)
    args["max_query"] = 90
    prefix_attention(**args, out=out, lse=lse)
    for part in (slice(0, 3), slice(163, 165)):
        assert not out[part].any() and torch.isneginf(lse[part]).all()
    check(b, out[3:163], lse[3:163], None, want)


def test_no_slots_at_all():
    b = Batch([0, 0], counts=[40, 33], heads=1, group=2, seed=16)
    args = b.on_gpu()
    args.update(table=args["table"][:, :0])
    out, lse = prefix_attention(**args)
    assert not out.any() and torch.isneginf(lse).all()
    args.update(kv_cache=args["kv_cache"][:0])
    out, lse = prefix_attention(**args)
    assert not out.any() and torch.isneginf(lse).all()


@pytest.mark.parametrize("scale", [0.25, -0.25, 0.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=lambda t: str(t)[6:])
def test_growing_logits(dtype, scale):
    # the maximum of a query moves on with every key, in steps below and above what the running maximum is kept over
    b = Batch([400], counts=[70], prefixes=[90], heads=1, group=1, dim=32, dtype=dtype, seed=17).with_scores()
    b.query.abs_()
    flat = torch.linspace(0.05, 3.0, 490).repeat_interleave(1)
    order = [*b.prefix_table[0, : -(-90 // 16)], *b.table[0, : -(-400 // 16)]]
    at = 0
    for part, n in ((order[: -(-90 // 16)], 90), (order[-(-90 // 16):], 400)):
        for j in range(n):
            b.cache[int(part[j // 16]), 0, j % 16] = (flat[at] * (1 + 0.01 * torch.randn(1, 32))).to(dtype)
            at += 1
    b.scale = scale
    check(b, *run(b))


def test_one_key_takes_all_the_weight():
    b = Batch([300], counts=[80], prefixes=[100], heads=1, group=2, spread=400.0, seed=18)
    out, lse, _ = run(b)
    want = b.want()
    assert torch.isfinite(out).all()
    gap = np.abs(lse.double().cpu().numpy() - want["lse"])
    assert np.all(gap <= 2 * (b.dim + 4) * 2.0**-24 * want["reach"] + 1e-5)


def test_equal_calls_give_equal_bits():
    b = Batch([300, 75, 2000], counts=[74, 74, 90], prefixes=[700], heads=2, group=3, seed=20).with_scores()
    first = run(b)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, run(b)))


@pytest.mark.parametrize("counts", [[70, 66], [1, 1]])
def test_graph_replays(counts):
    rows = 2 if counts[0] > 1 else 40
    b = Batch([100 + r for r in range(rows)], counts=(counts * rows)[:rows], prefixes=[270], heads=1, group=4, seed=22)
    b.with_scores()
    args = b.on_gpu()
    start = args["scores"].clone()
    want_out, want_lse = prefix_attention(**args)
    want_scores = args["scores"].clone()
    out, lse = torch.empty_like(want_out), torch.empty_like(want_lse)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            prefix_attention(**args, out=out, lse=lse)
    for _ in range(3):
        args["scores"].copy_(start)
        out.zero_()
        lse.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want_out) and torch.equal(lse, want_lse) and torch.equal(args["scores"], want_scores)
        prefix_attention(**b.on_gpu())
        torch.cuda.synchronize()


@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_weights_of_many_query_rows(dtype, dim):
    # 600 query rows a KV head, few rows: the weights of 64 keys are a workgroup's
    b = Batch([170, 90], counts=[150, 90], prefixes=[37], heads=1, group=4, dim=dim, dtype=dtype, seed=dim + 2).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("block", [16, 24])
def test_weights_behind_bad_pages(block):
    b = Batch([170, 130, 0], counts=[150, 129, 0], heads=1, group=4, block=block, seed=21).with_scores()
    b.table[0, 1], b.table[0, 3], b.table[1, :] = -1, b.cache.shape[0], 2**31 - 1
    check(b, *run(b))


@pytest.mark.parametrize("queries", [4, 5, 16, 17])
@pytest.mark.parametrize("dim", [64, 256])
def test_around_the_wide_kernels_first_rows(queries, dim):
    b = Batch([90, 33, 200], counts=[queries, 1, queries], prefixes=[70], heads=1, group=4, dim=dim, seed=queries).with_scores()
    check(b, *run(b))
    b = Batch([30 + r for r in range(2 * queries)], prefixes=[70, 90], borders=[0, queries, 2 * queries], heads=1, group=4,
              dim=dim, seed=queries)
    check(b, *run(b))


@pytest.mark.parametrize("counts", [[1], [70]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=lambda t: str(t)[6:])
def test_small_weights_beside_one_large(dtype, counts):
    # one key holds nearly all the weight, the others 2^-27 of it each, with values that matter all the same
    b = Batch([600], counts=counts, prefixes=[200], heads=1, group=1, dim=32, dtype=dtype, seed=23)
    b.cache[:, 0], b.query[:] = 0.0, 0.0
    b.query[..., 0] = 27 * np.log(2.0)
    b.scale = 1.0
    b.cache[:, 1] = 200.0
    page = int(b.prefix_table[0, 0])
    b.cache[page, 0, 3, :, 0] = 1.0
    b.cache[page, 1, 3] = 2.0**-10
    check(b, *run(b))


@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_a_prompt_among_single_tokens(dtype):
    counts = [1] * 90
    counts[7], counts[40], counts[41] = 300, 0, 66
    b = Batch([max(n, 20 + r) for r, n in enumerate(counts)], counts=counts, prefixes=[50, 30], borders=[3, 41, 80], heads=1,
              group=2, dim=32, dtype=dtype, seed=24).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("ends", [(0, 0), (1, 0), (0, 2)])
def test_tokens_of_no_row_beside_a_prompt_among_single_tokens(ends):
    # 70 rows, the first and the last maybe without queries
    counts = [ends[0]] + [1] * 30 + [300] + [1] * 37 + [ends[1]]
    b = Batch([max(n, 20 + r) for r, n in enumerate(counts)], counts=counts, heads=1, group=2, dim=32, seed=25)
    tokens = sum(counts)
    want = b.want()
    b.max_query = 299  # the prompt's last query is past it
    bounded = b.want()
    args = b.on_gpu()
    query = torch.randn(5 + tokens + 3, 2, 32, dtype=torch.bfloat16, device="cuda")
    query[5 : 5 + tokens] = args["query"]
    args.update(query=query, q_start=args["q_start"] + 5)
    for most, expected in ((299, bounded), (300, want)):
        out, lse = torch.full_like(query, 9.0), torch.full((8 + tokens, 2), 9.0, device="cuda")
        prefix_attention(**dict(args, max_query=most), out=out, lse=lse)
        for part in (slice(0, 5), slice(5 + tokens, 8 + tokens)):
            assert not out[part].any() and torch.isneginf(lse[part]).all()
        check(b, out[5 : 5 + tokens], lse[5 : 5 + tokens], None, expected)
