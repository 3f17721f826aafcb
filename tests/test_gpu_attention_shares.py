"""Decode attention's equal shares of all rows' keys: many rows, rows of nothing between them, one row across every
wave, more heads and tiles than waves, lengths at the borders of steps and shares; against the definition in float64."""

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


@pytest.mark.parametrize("rows", [255, 256, 257, 700])
def test_many_rows(rows):
    b = Batch([(r * 37) % 90 if r % 5 else 0 for r in range(rows)], heads=1, group=2, dim=32, seed=rows).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_one_long_row_among_short_ones(dtype):
    b = Batch([3, 0, 9000, 1, 64, 0], heads=1, group=1, dim=32, dtype=dtype, seed=2).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float8_e4m3fn, 256), (torch.float32, 128)])
def test_a_row_in_as_many_slots_as_there_are(dtype, dim):
    b = Batch([6000], heads=1, group=1, dim=dim, dtype=dtype, seed=3).with_scores()
    check(b, *run(b))


def test_more_heads_and_tiles_than_waves():
    # 90 KV heads of 33 query heads: three tiles each, 270 pairs of head and tile
    b = Batch([40, 7], heads=90, group=33, dim=32, seed=4).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("length", [15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 1023, 1024, 1025])
def test_lengths_at_borders(length):
    b = Batch([length, length + 1, 1, length], heads=1, group=2, dim=64, seed=length).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("counts", [[2, 2, 2, 2], [5, 1, 0, 3], [1, 40, 7, 16]])
def test_a_few_queries_a_row(counts):
    # queries of a row that see nothing of its last pieces, tiles that a row does not have
    b = Batch([2, 600, 33, 1500], counts=counts, heads=2, group=1, dim=32, seed=6).with_scores()
    check(b, *run(b))


@pytest.mark.parametrize("rows,queries", [(40, 1), (300, 4)])
def test_joins_of_few_and_many_queries(rows, queries):
    b = Batch([50 + r % 40 for r in range(rows)], counts=[queries] * rows, prefixes=[900], heads=1, group=2, dim=32, seed=7)
    check(b, *run(b))


def test_tables_of_the_most_keys():
    # the table is wide enough for lengths near 2^31; the row is short
    b = Batch([70], heads=1, group=2, dim=32, seed=8)
    args = b.on_gpu()
    need = args["table"].shape[1]
    wide = torch.full((1, (2**31 - 4096) // 16 - 1), -1, dtype=torch.int32, device="cuda")
    wide[:, :need] = args["table"]
    out, lse = prefix_attention(**dict(args, table=wide))
    check(b, out, lse)
