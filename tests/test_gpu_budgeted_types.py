"""With a rotation BudgetedCache takes the types and strides that it takes without."""

import pytest
import torch

from runtime.budgeted_cache import BudgetedCache
from runtime.rotary import rotary_frequencies

pytestmark = pytest.mark.gpu
F32, F16, BF16, FP8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
ROWS, HEADS, GROUP, DIM = 3, 2, 2, 32


def caches_of(dtype, weights, count=2):
    turn = dict(frequencies=rotary_frequencies(DIM // 2))
    if weights is not None:
        turn.update(q_weight=torch.linspace(0.5, 1.5, DIM, device="cuda").to(weights),
                    k_weight=torch.linspace(1.5, 0.5, DIM, device="cuda").to(weights))
    scale = 0.02 if dtype == FP8 else 1.0
    return [BudgetedCache(ROWS, HEADS, DIM, budget=24, slack=8, prefix=5, block=4, dtype=dtype, k_scale=scale, v_scale=scale,
                          rotation=turn) for _ in range(count)]


def same(a, b):
    assert torch.equal(a.kv.view(torch.uint8), b.kv.view(torch.uint8))
    for name in ("lens", "seen", "positions", "scores", "prefix_len"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    assert a.longest == b.longest


def projected(n):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(n)
    x = torch.randn(n, HEADS * (GROUP + 2), DIM, generator=gen, device="cuda", dtype=torch.float64)
    return x[:, :HEADS * GROUP], x[:, HEADS * GROUP:HEADS * (GROUP + 1)], x[:, HEADS * (GROUP + 1):]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("given", [F32, F16, BF16, torch.float64], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("weights", [None, F32])
def test_types_are_rounded_to_the_caches(dtype, given, weights):
    a, b = caches_of(dtype, weights)
    _, keys, values = (x.to(given) for x in projected(4))
    a.set_prefix(keys, values)
    b.set_prefix(keys.to(dtype), values.to(dtype))
    start = torch.tensor([0, 2, 2, 7], device="cuda")
    for n, q_start, most in ((7, start, 5), (ROWS, None, 1)):
        query, keys, values = (x.to(given) for x in projected(n))
        got = a.append(keys, values, q_start, most, query=query)
        want = b.append(keys.to(dtype), values.to(dtype), q_start, most, query=query.to(dtype))
        assert got.dtype == dtype and torch.equal(got, want)
    a.append(keys, values.to(BF16))
    b.append(keys.to(dtype), values.to(BF16).to(dtype))
    same(a, b)


@pytest.mark.parametrize("types", [(BF16, F32, F32), (BF16, BF16, F32), (F32, torch.float64, F16), (BF16, BF16, FP8)],
                         ids=lambda ts: "-".join(str(t)[6:] for t in ts))
@pytest.mark.parametrize("weights", [None, BF16, F32])
def test_an_fp8_cache_takes_mixed_types(types, weights):
    """They meet in float32; the queries come back of their own type, as the attention takes them."""
    a, b = caches_of(FP8, weights)
    if weights is not None:
        b.rotation = {**b.rotation, **{k: b.rotation[k].float() for k in ("q_weight", "k_weight")}}
    _, keys, values = (x.to(t) for x, t in zip(projected(4), types))
    a.set_prefix(keys, values)
    b.set_prefix(keys.float(), values.float())
    query, keys, values = (x.to(t) for x, t in zip(projected(ROWS), types))
    got = a.append(keys, values, query=query)
    want = b.append(keys.float(), values.float(), query=query.float())
    assert got.dtype == types[0] and torch.equal(got, want.to(types[0]))
    same(a, b)
    if types[0] == BF16:
        a.attend(got, DIM**-0.5)


@pytest.mark.parametrize("dtype", [F32, BF16, FP8], ids=lambda t: str(t)[6:])
def test_views_of_any_alignment(dtype):
    kind = BF16 if dtype == FP8 else dtype
    a, b = caches_of(dtype, None)

    def off(x):  # the same values, off 16 bytes
        wide = torch.zeros(*x.shape[:2], DIM + 1, dtype=x.dtype, device="cuda")
        wide[..., 1:] = x
        return wide[..., 1:]

    def apart(x):  # elements apart
        return torch.stack([x, x], -1)[..., 0]

    for view in (off, apart):
        query, keys, values = (x.to(kind) for x in projected(ROWS))
        got = a.append(view(keys), view(values), query=view(query))
        assert torch.equal(got, b.append(keys, values, query=query))
        same(a, b)
    _, keys, values = (x.to(kind) for x in projected(5))
    a.set_prefix(off(keys), apart(values))
    b.set_prefix(keys, values)
    same(a, b)
