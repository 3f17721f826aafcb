"""A query of NaN: its own output and the scores of the keys it sees are NaN, nothing else changes."""

import pytest
import torch

from attention_cases import Batch
from runtime.prefix_attention import prefix_attention

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float32]


@pytest.mark.parametrize("group", [2, 12])  # the kept logits; more than 16 query rows a KV head: the keys read again
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_keys_it_does_not_see_keep_their_scores(dtype, group):
    b = Batch([39, 23, 2], counts=[2, 2, 2], heads=2, group=group, dtype=dtype, seed=3).with_scores()
    b.table[0, 1] = -1  # slots 16 to 31 of the first row are not there
    clean = b.on_gpu()
    out, lse = prefix_attention(**clean)
    args = b.on_gpu()
    args["query"][0] = float("nan")  # the first row's first query
    got_out, got_lse = prefix_attention(**args)
    torch.cuda.synchronize()
    assert torch.isnan(got_out[0]).all() and torch.isnan(got_lse[0]).all()
    assert torch.equal(got_out[1:], out[1:]) and torch.equal(got_lse[1:], lse[1:])
    scores, want = args["scores"], clean["scores"]
    assert torch.equal(scores[1:], want[1:])
    seen = [j for j in range(38) if not 16 <= j < 32]
    assert torch.isnan(scores[0, :, seen]).all()
    others = [j for j in range(scores.shape[2]) if j not in seen]
    assert torch.equal(scores[0][:, others], want[0][:, others])
