"""Token eviction at the sizes where its kernel changes form: rows up to 2048, 4096, 6144, 8192, 16384 slots and longer,
few and many rows; ties, special scores, odd capacities and buffers in place. All exact."""

import numpy as np
import pytest
import torch

from test_gpu_eviction import batch, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("length", [2047, 2048, 2049, 4095, 4097, 6100, 6145, 8192, 8200, 16384, 16390])
def test_capacities(length, in_place):
    b = batch([length, length // 3, 1], heads=1, seed=length, room=0)
    run(b, [length // 2, 7, 1], [length, length // 3, 1], in_place, recent=20, sinks=4)
    b = batch([length, length - 1, 5], heads=1, seed=length + 1, ties=True, room=1)
    run(b, [length - 3, length // 2, 9], [length, length - 1, 5], in_place)


@pytest.mark.parametrize("block,length", [(1, 2049), (3, 4001), (7, 8190), (24, 9000)])
def test_capacities_that_are_no_multiple_of_four(block, length):
    b = batch([length, 70], heads=2, block=block, seed=block, ties=True, room=0)
    for in_place in (False, True):
        run(b, [length - 1, 33], [length, 70], in_place, recent=9)


@pytest.mark.parametrize("length", [300, 3000, 5000, 7000, 12000])
def test_equal_scores_and_specials(length):
    b = batch([length], heads=1, seed=length)
    b[3][:] = 0.0
    run(b, [length // 2], [length], sinks=2)
    rng = np.random.default_rng(1)
    b[3][:] = rng.choice([np.nan, -np.inf, np.inf, -0.0, 0.0, 1e-45, -1e-45, 3e38, 1.0, np.float32(1.0000001)],
                         size=b[3].shape)
    for budget in (1, length // 3, length - 1):
        run(b, [budget], [length], recent=length // 10)


def test_more_rows_than_compute_units():
    # every workgroup copies its own moves
    lens = [40 + (r * 13) % 90 for r in range(520)]
    run(batch(lens, heads=1, seed=2), [n // 2 for n in lens], lens, recent=4, sinks=1)


def test_few_rows_that_move_much():
    # the moves are listed and spread over the chip
    run(batch([9000, 8500], heads=1, dim=256, dtype=torch.float32, seed=3), [4000, 4200], [9000, 8500], recent=64)


def test_bad_pages_in_both_forms():
    for lens, dim, dtype in (([100, 64], 32, torch.bfloat16), ([9000], 256, torch.float32)):
        b = batch(lens, heads=1, dim=dim, dtype=dtype, seed=4)
        b[1][0, 1], b[1][0, 5] = -1, b[0].shape[0]
        run(b, [n // 2 for n in lens], lens)
