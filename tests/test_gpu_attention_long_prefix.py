"""A prefix of more than 2^30 tokens: few pages, listed again and again."""

import math

import pytest
import torch

from runtime.prefix_attention import prefix_attention


@pytest.mark.gpu
def test_prefix_past_a_billion_tokens():
    # 1029 times a page of logit 0 and value 1, then 5 tokens of logit 60 and value 2, which outweigh 2^30 times exp(0)
    block, pages = 1 << 20, 1030
    cache = torch.zeros(4, 2, block, 1, 32, device="cuda").to(torch.float8_e4m3fn)
    raw = cache.view(torch.uint8)
    code = {x: int(torch.tensor(x).to(torch.float8_e4m3fn).view(torch.uint8)) for x in (1.0, 2.0, 7.5)}
    raw[1, 1] = code[1.0]
    raw[2, 1] = code[2.0]
    raw[2, 0, :, :, 0] = code[7.5]
    query = torch.zeros(1, 1, 32, dtype=torch.bfloat16, device="cuda")
    query[..., 0] = 8.0
    table = torch.full((1, pages), 1, dtype=torch.int32, device="cuda")
    table[0, -1] = 2
    lens = torch.tensor([(pages - 1) * block + 5], dtype=torch.int32, device="cuda")
    own = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    out, lse = prefix_attention(query, cache, own, own[0], 1.0, prefix_table=table, prefix_lens=lens)
    assert torch.all(out == 2.0), out
    # the logits and the sum are exact here: the rest is the logarithm and the sum of two terms
    assert abs(lse.item() - (60.0 + math.log(5.0))) <= 8 * 2.0**-24 * 62.0
