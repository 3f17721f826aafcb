"""Which keys are read together, told on the host by the workspace: a prefix read once for its group leaves partial results
that are joined to the rows' own, a row's tile that walks prefix and own keys in one pass leaves none."""

import ctypes

import ekv_hip
from test_attention_refusals import P, attention


def slots(rows, max_query, tokens, prefix, groups=1, width=38, **over):
    """Partial results that the workspace has room for, a query's."""
    a = attention(**{**dict(rows=rows, width=width, table_stride=width, tokens=tokens, max_query=max_query, q_start=P,
                            prefix_table=P, prefix_lens=P, prefix_rows=P, prefix_groups=groups, prefix_width=prefix // 16,
                            prefix_stride=prefix // 16, q_heads=32, kv_heads=8, head_dim=128), **over})
    need = ekv_hip.load().ekv_prefix_attention_workspace(ctypes.addressof(a))
    assert need > 0
    return need // (tokens * a.q_heads * (a.head_dim * 4 + 8))


def test_few_queries_share_their_prefix():
    for queries in (1, 2, 4, 5, 8, 16):  # 4 to 64 query rows a KV head and row
        assert slots(200, queries, 200 * queries, 32768, groups=2) >= 2
    assert slots(128, 2, 256, 8192, q_heads=128) >= 2  # 2 tokens of 16 heads a KV head
    assert slots(128, 20, 128 * 20, 32768, q_heads=8) >= 2
    assert slots(64, 20, 64 * 20, 32768, head_dim=256) >= 2


def test_a_prompt_among_single_tokens_shares_its_prefix():
    assert slots(128, 2048, 2048 + 127, 8192, width=128) >= 2


def test_rows_that_fill_their_tiles_walk_their_prefix_in_one_pass():
    assert slots(5, 1024, 5 * 700, 1999 // 16 * 16, width=188) == 0
    assert slots(64, 64, 64 * 64, 32768) == 0
    assert slots(128, 5, 128 * 5, 64) == 0  # nothing to save by a prefix of 64 tokens


def test_kept_logits_fit_a_launch():
    """Folding the kept logits takes a workgroup of 256 for every (row, KV head), however short the row: from 2^24 of them on
    that is no launch, and the weights are computed from the keys again."""
    def more(rows):  # bytes that the scores add to the workspace
        sizes = []
        for scores in (0, P):
            a = attention(rows=rows, tokens=rows, q_heads=8, kv_heads=8, head_dim=32, width=1, table_stride=1, block_size=16,
                          scores=scores, scores_stride_row=128, scores_stride_head=16)
            sizes.append(ekv_hip.load().ekv_prefix_attention_workspace(ctypes.addressof(a)))
            assert sizes[-1] > 0
        return sizes[1] - sizes[0]

    kept = (1 << 21) - 1  # rows of 8 KV heads
    assert more(kept) == kept * 8 * 16 * 4
    assert more(1 << 21) == 0
