"""The rows of an append's tokens at the edges of their search, and launches of more waves than threads allow."""

import numpy as np
import pytest
import torch

from append_cases import Tokens, check
from runtime.append import append_tokens
from runtime.rotary import rotary_frequencies

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("rows", [253, 254, 255, 256, 257, 16256, 16257, 16300, 20000])
@pytest.mark.parametrize("empty", [False, True])
def test_rows_at_the_edges_of_the_search(rows, empty):
    """A wave's window holds 254 starts; of more rows it first narrows them 64 times, of more than 16256 twice.  ``empty``: runs of
    empty rows at both ends and across the starts that it narrows by."""
    rng = np.random.default_rng(rows)
    counts = rng.integers(0, 3, size=rows)
    counts[0] = counts[-1] = 2
    if empty:
        step = -(-rows // 64)
        for probe in range(step - 1, rows, 3 * step):
            counts[max(0, probe - 2):probe + 3] = 0
        counts[:3] = counts[-3:] = 0
    batch = Tokens(counts + 1, counts, q_heads=1, kv_heads=1, dim=16, block=4, ahead=2, behind=3, seed=31)
    args = batch.on_gpu()
    check(batch, args, append_tokens(**args))


@pytest.mark.parametrize("tokens", [2**24 + 5, 2**25 + 7])
def test_passes_enough_for_waves_that_a_launch_has_not(tokens):
    """Six passes a token would take four waves, or two, where 2^32 threads leave two and one.  Five rows keep 20 tokens each, read
    from one row of keys and told apart by their positions; the rest belongs to nobody's slots."""
    heads, dim, block, most = 9, 256, 16, 20
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    one = torch.randn(2, 1, heads, dim, generator=gen, device="cuda").to(BF16)
    keys, values = one[0].expand(tokens, heads, dim), one[1].expand(tokens, heads, dim)
    starts = [0, 31, 2**22 - 3, 2**23 + 9, tokens - 12, tokens]
    at = torch.arange(tokens, dtype=torch.int32, device="cuda")
    f = rotary_frequencies(dim // 2)
    table = torch.arange(10, dtype=torch.int32, device="cuda").view(5, 2)
    got, want = (torch.zeros(10, 2, block, heads, dim, dtype=BF16, device="cuda") for _ in range(2))
    lens = torch.zeros(5, dtype=torch.int32, device="cuda")
    append_tokens(got, table, lens, keys, values, q_start=torch.tensor(starts, dtype=torch.int32, device="cuda"), max_query=most,
                  positions=at, frequencies=f, advance=True)
    kept = [min(most, b - a) for a, b in zip(starts, starts[1:])]
    assert lens.tolist() == kept == [20, 20, 20, 20, 12]
    for r, n in enumerate(kept):
        a = starts[r]
        append_tokens(want, table[r:r + 1], torch.zeros(1, dtype=torch.int32, device="cuda"), keys[:n], values[:n],
                      q_start=torch.tensor([0, n], dtype=torch.int32, device="cuda"), max_query=n, positions=at[a:a + n],
                      frequencies=f, advance=True)
    assert torch.equal(got, want)
