"""Logits far apart, and at the type's lowest value: the outputs, not only that they are finite."""

import numpy as np
import pytest
import torch

from attention_cases import Batch, check
from runtime.prefix_attention import prefix_attention

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float32]
SHAPES = {  # single tokens, drafts, prompts, rows of some queries behind a prefix table wide enough to share it
    "tokens": dict(lens=[200, 40, 133], counts=None, prefixes=[90]),
    "drafts": dict(lens=[200, 40, 133], counts=[3, 1, 4], prefixes=[90]),
    "prompts": dict(lens=[200, 140], counts=[130, 100], prefixes=[90]),
    "together": dict(lens=[60, 140, 80, 90], counts=[12, 20, 10, 9], prefixes=[90]),
}


def batch(shape, dtype, **more):
    b = Batch(**SHAPES[shape], heads=2, group=2, dtype=dtype, **more).with_scores()
    if shape == "together":
        table = np.full((1, (1 << 20) // b.block), -1, np.int32)
        table[:, : b.prefix_table.shape[1]] = b.prefix_table
        b.prefix_table = table
    return b


def run(b):
    args = b.on_gpu()
    out, lse = prefix_attention(**args)
    torch.cuda.synchronize()
    return out, lse, args["scores"]


def slots(b):
    """(page, slot) of every cached token, prefix and rows each in their order."""
    for pages, n in [*zip(b.table, b.lens), (b.prefix_table[0], b.prefix_lens[0])]:
        for j in range(int(n)):
            yield int(pages[j // b.block]), j % b.block, j


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_one_key_wins_by_far(dtype, shape):
    # A key's only element is its number over the dims, counted up from 1 for the own tokens and from 1/2 for the prefix's;
    # a query has one element, so the last seen key of that dim is 128 or more ahead: the others' weights are below
    # 2^-184, nothing beside it in float32, and the output is its value row, bit for bit.
    b = batch(shape, dtype, seed=41)
    b.k_scale = b.v_scale = 1.0
    b.scale = 1.0
    b.cache[:, 0] = torch.zeros_like(b.cache[:, 0])
    b.cache[:, 1] = torch.randn(b.cache[:, 1].shape, generator=torch.Generator().manual_seed(2)).to(dtype)
    raw = b.cache.float()
    prefix = set(b.prefix_table[0, : -(-90 // b.block)].tolist())
    for page, slot, j in slots(b):
        raw[page, 0, slot, :, j % b.dim] = j // b.dim + (0.5 if page in prefix else 1.0)
    b.cache = raw.to(dtype)
    b.query[:] = 0.0
    for t in range(b.query.shape[0]):
        b.query[t, :, (5 * t + 3) % 30] = 256.0  # every query sees a key of these dims: the prefix has all
    want = b.want()
    out, lse, scores = run(b)
    check(b, out, lse, scores, want)
    assert torch.equal(out.cpu(), torch.from_numpy(want["out"]).to(out.dtype))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_logits_far_apart(dtype, shape):
    b = batch(shape, dtype, seed=42, spread=400.0)
    check(b, *run(b))


@pytest.mark.parametrize("counts", [[1], [40]], ids=["token", "prompt"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=lambda t: str(t)[6:])
def test_equal_weights_at_the_lowest_value(dtype, counts):
    # every logit is half the type's lowest value, so a query's output is the mean of the values that it sees
    b = Batch([40], counts=counts, heads=1, group=4, dtype=dtype, seed=43).with_scores()
    b.query[:] = 1.0
    b.cache[:, 0] = torch.finfo(dtype).min / 128
    b.scale = 1.0
    out, lse, scores = run(b)
    t = counts[0]
    values = np.stack([b.cache[int(b.table[0, j // 16]), 1, j % 16, 0].double().numpy() for j in range(40)])
    added = np.zeros(40)
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    for i in range(t):
        seen = 40 - t + i + 1
        added[:seen] += b.group / seen
        mean, size = values[:seen].mean(axis=0), np.abs(values[:seen]).mean(axis=0)
        # weights of one are exact in every type; sum and mean in float32, then the output's rounding
        bound = (seen + 64) * 2.0**-24 * size + max(half, 2.0**-24) * np.abs(mean)
        assert np.all(np.abs(out[i].double().cpu().numpy() - mean) <= bound)
    assert torch.isfinite(lse).all()
    # a key's weight is exp(s - lse), and lse at this size holds log(seen) to half a step of float32 at best
    if dtype == torch.float16:
        old = b.scores[0, 0, :40].double().numpy() * b.decay
        off = np.abs(scores[0, 0, :40].double().cpu().numpy() - old - added)
        step = 2.0**-24 * 32752 * 4  # of s and lse: their products with log2(e), their difference
        assert np.all(off <= (step + 128 * 2.0**-24) * added + 2.0**-23 * (old + added))


@pytest.mark.parametrize("scale", [-3e31, -1e9, -40.0, 0.1, 3.0, 7.0, 19.0, 83.0, 1e3, 1e7, 3e31])
@pytest.mark.parametrize("counts", [None, [40, 70]], ids=["tokens", "prompts"])
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_equal_weights_of_every_size(dtype, counts, scale):
    # equal logits of scale * 2^20 or so, up to 2^125: the outputs stay the mean of the values that are seen
    b = Batch([40, 90], counts=counts, prefixes=[21], heads=1, group=2, dtype=dtype, seed=44)
    b.k_scale = b.v_scale = 1.0
    b.cache[:, 0], b.query[:] = 120.0, 140.0
    b.scale = scale
    out, lse, _ = run(b)
    half = 0.0 if dtype == torch.float32 else torch.finfo(out.dtype).eps / 2
    shared = [b.cache[int(b.prefix_table[0, j // 16]), 1, j % 16, 0].double().numpy() for j in range(21)]
    token = 0
    for r, n in enumerate(b.lens):
        values = np.stack(shared + [b.cache[int(b.table[r, j // 16]), 1, j % 16, 0].double().numpy() for j in range(n)])
        t = 1 if counts is None else counts[r]
        for i in range(t):
            seen = 21 + n - t + i + 1
            mean, size = values[:seen].mean(axis=0), np.abs(values[:seen]).mean(axis=0)
            # as above, and a half step for a weight's rounding
            bound = ((seen + 64) * 2.0**-24 + half) * size + max(half, 2.0**-24) * np.abs(mean)
            assert np.all(np.abs(out[token].double().cpu().numpy() - mean) <= bound), (r, i)
            token += 1
    assert torch.isfinite(lse).all()


@pytest.mark.parametrize("scale", [-3e31, -1e9, -40.0, 7.0, 83.0, 1e3, 1e7, 3e31])
@pytest.mark.parametrize("counts,group", [(None, 2), ([9, 9], 2), ([40, 70], 2), ([140, 150], 4)],
                         ids=["kept", "again", "wide", "workgroups"])
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_a_weight_is_at_most_one(dtype, counts, group, scale):
    # float32's steps of such logits are whole powers of two: what a weight is, its lse cannot say, but no more than 1
    b = Batch([180, 190], counts=counts, prefixes=[21], heads=1, group=group, dtype=dtype, seed=45).with_scores()
    b.k_scale = b.v_scale = 1.0
    b.cache[:, 0], b.query[:] = 120.0, 140.0
    b.scale = scale
    old = b.scores.double().numpy()
    _, _, scores = run(b)
    got, queries = scores.double().cpu().numpy(), b.max_query * group
    for r, n in enumerate(b.lens):
        held = old[r, :, :n] * b.decay
        slack = (queries + 8) * 2.0**-24 * (held + queries)  # of as many additions
        assert np.all(got[r, :, :n] >= held - slack) and np.all(got[r, :, :n] <= held + queries + slack)
        assert np.array_equal(got[r, :, n:], old[r, :, n:])
