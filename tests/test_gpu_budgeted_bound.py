"""What BudgetedCache.append takes on the GPU."""

import pytest
import torch

from runtime.budgeted_cache import BudgetedCache

pytestmark = pytest.mark.gpu
BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn
ROWS, HEADS, DIM = 3, 2, 32


@pytest.mark.parametrize("dtype", [BF16, FP8], ids=lambda t: str(t)[6:])
def test_a_bound_above_one_without_starts(dtype):
    """A token a row, whatever the bound; the host counts by the bound."""
    caches = [BudgetedCache(ROWS, HEADS, DIM, budget=8, slack=8, block=4, dtype=dtype, device=d) for d in ("cuda", "cpu")]
    gen = torch.Generator().manual_seed(1)
    for step in range(4):
        rows = torch.randn(ROWS, HEADS, DIM, generator=gen)
        for c in caches:
            c.append(rows.to(c.kv.device), -rows.to(c.kv.device), max_query=3)
    here, host = caches
    assert here.longest == host.longest == 12
    for name in ("lens", "seen", "positions", "scores"):
        assert torch.equal(getattr(here, name).cpu(), getattr(host, name)), name
    assert torch.equal(here.kv.cpu()[1:].view(torch.uint8), host.kv[1:].view(torch.uint8))
