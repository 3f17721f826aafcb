"""Norms of heads whose squares leave float32: small elements with an eps of 0 or next to it, large ones with small weights."""

import numpy as np
import pytest
import torch

from append_cases import bound
from runtime.append import append_tokens
from runtime.rotary import rotate_heads

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DIM = 64


def normed(x, weight, eps):
    wide = x.double().cpu().numpy()
    return wide / np.sqrt((wide * wide).mean(-1, keepdims=True) + float(np.float32(eps))) * weight.double().cpu().numpy()


def close(got, want, dtype):
    off = np.abs(got.double().cpu().numpy() - want)
    assert np.all(off <= bound(want, np.abs(want), dtype, DIM, True, 0.0, False)), off.max()


def seeded(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def heads(tokens, count, sizes, dtype, seed=1):
    """Token t's elements are of size ``sizes[t % len(sizes)]``."""
    gen = seeded(seed)
    size = torch.tensor(sizes, dtype=torch.float64, device="cuda")[torch.arange(tokens, device="cuda") % len(sizes)]
    return (torch.randn(tokens, count, DIM, generator=gen, device="cuda", dtype=torch.float64) * size[:, None, None]).to(dtype)


SMALL = [1.0, 1e-15, 1e-18, 3e-19, 1e-20, 3e-22, 1e-24, 1e-30, 1e-37, 1e-39]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("eps", [0.0, 1e-41, 1e-38, 1e-34, 1e-30, 1e-20])
@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("tokens,count", [(20, 5), (8200, 1)])  # the second: several tokens a wave
def test_small_elements(dtype, eps, own, tokens, count):
    x = heads(tokens, count, SMALL, dtype)
    w = 1 + 0.3 * torch.randn((count, DIM) if own else (DIM,), generator=seeded(5), device="cuda")
    got, _ = rotate_heads(x, None, None, None, q_weight=w, eps=eps)
    close(got, normed(x, w, eps), dtype)


@pytest.mark.parametrize("eps", [0.0, 1e-41])
def test_heads_of_zeros_beside_small_ones(eps):
    """0 / 0 with an eps of 0, else 0; the heads beside are their own."""
    x = heads(6, 2, [1e-24], F32)
    x[2] = 0
    x[4, 1] = 0
    w = torch.ones(DIM, device="cuda")
    got, _ = rotate_heads(x, None, None, None, q_weight=w, eps=eps)
    zero = (x == 0).all(-1)
    assert torch.all(torch.isnan(got[zero]) if eps == 0 else got[zero] == 0)
    close(got[~zero], normed(x[~zero], w, eps), F32)


def test_single_elements_and_one_that_is_not_finite():
    x = torch.zeros(4, 1, DIM, device="cuda")
    x[0, 0, 9] = 2.0**-149
    x[1, 0, 50] = -3e-23
    x[2, 0, :] = 1e-25
    x[2, 0, 3] = float("nan")
    x[3, 0, :] = 1e-25
    x[3, 0, 3] = float("inf")
    w = torch.ones(DIM, device="cuda")
    got, _ = rotate_heads(x, None, None, None, q_weight=w, eps=0.0)
    close(got[:2], normed(x[:2], w, 0.0), F32)
    assert torch.all(torch.isnan(got[2])) and torch.isnan(got[3, 0, 3])
    assert torch.all(got[3, 0, torch.arange(DIM, device="cuda") != 3] == 0)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: str(t)[6:])
def test_keys_on_their_way_into_a_cache(dtype):
    tokens, block = 20, 16
    x = heads(tokens, 2, SMALL, dtype, 2)
    w = 1 + 0.3 * torch.randn(DIM, generator=seeded(5), device="cuda")
    cache = torch.zeros(tokens, 2, block, 2, DIM, dtype=dtype, device="cuda")
    table = torch.arange(tokens, dtype=torch.int32, device="cuda").view(tokens, 1)
    one = torch.ones(tokens, dtype=torch.int32, device="cuda")
    query = append_tokens(cache, table, one, x, x, query=x, q_weight=w, k_weight=w, eps=0.0)
    want = normed(x, w, 0.0)
    close(query, want, dtype)
    close(cache[:, 0, 0], want, dtype)
    assert torch.equal(cache[:, 1, 0], x)

@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("weight", [1.0, 1e-2, 1e-4, 1e-8])
@pytest.mark.parametrize("tokens,count", [(12, 3), (8200, 1)])
def test_large_elements_with_small_weights(dtype, weight, tokens, count):
    x = heads(tokens, count, [1.0, 2.0**64, 2.0**90, 2.0**110, 2.0**124], dtype, 3).clamp(-3e38, 3e38)
    w = weight * (1 + 0.3 * torch.rand(DIM, generator=seeded(5), device="cuda"))
    got, _ = rotate_heads(x, None, None, None, q_weight=w, eps=1e-6)
    close(got, normed(x, w, 1e-6), dtype)
    mixed = x.clone()  # small elements beside large ones
    mixed[..., ::2] *= 2.0**-60
    got, _ = rotate_heads(mixed, None, None, None, q_weight=w, eps=1e-6)
    close(got, normed(mixed, w, 1e-6), dtype)
