"""What the attention and eviction calls refuse, on the host: the C ABI's checks (which need no GPU) and the
Python layer's."""

import ctypes

import pytest
import torch

import ekv_hip
from runtime.eviction import evict_tokens
from runtime.prefix_attention import prefix_attention

P = 4096  # a placeholder device address: the checks refuse the call before using it


def attention(**over):
    a = ekv_hip.Attention()
    base = dict(query=P, q_stride_token=512, q_stride_head=64, keys=P, values=P, kv_stride_block=4096,
                kv_stride_pos=128, kv_stride_head=64, blocks=10, table=P, table_stride=4, lens=P, out=P,
                out_stride_token=512, out_stride_head=64, lse=P, q_dtype=ekv_hip.BF16, kv_dtype=ekv_hip.BF16, rows=3,
                width=4, tokens=3, max_query=1, q_heads=8, kv_heads=2, head_dim=64, block_size=16, scale=0.1,
                k_scale=1.0, v_scale=1.0, decay=1.0)
    for key, value in {**base, **over}.items():
        setattr(a, key, value)
    return a


@pytest.mark.parametrize("over,match", [
    (dict(q_dtype=ekv_hip.F16), "type"), (dict(kv_dtype=ekv_hip.F64), "type"),
    (dict(q_dtype=ekv_hip.FP8_E4M3, kv_dtype=ekv_hip.FP8_E4M3), "type"),
    (dict(q_dtype=ekv_hip.F16, kv_dtype=ekv_hip.FP8_E4M3), "type"),
    (dict(head_dim=96), "head dim"), (dict(head_dim=512), "head dim"), (dict(head_dim=0), "head dim"),
    (dict(q_heads=9), "heads"), (dict(kv_heads=0), "heads"), (dict(block_size=0), "block size"),
    (dict(rows=-1), "rows"), (dict(max_query=0), "queries"), (dict(tokens=4), "q_start"),
    (dict(max_query=2), "q_start"), (dict(width=1 << 27, block_size=16), "2\\^31"),
    (dict(prefix_groups=2, prefix_width=4, prefix_table=P, prefix_lens=P, prefix_stride=4), "prefix_rows"),
    (dict(prefix_groups=1, prefix_width=4, prefix_lens=P, prefix_stride=4), "null"),
    (dict(prefix_groups=1, prefix_width=4, prefix_table=P, prefix_lens=P, prefix_stride=3), "strides"),
    (dict(table_stride=3), "strides"), (dict(query=0), "null"), (dict(keys=0), "null"), (dict(lens=0), "null"),
    (dict(out=0), "null"), (dict(lse=0), "null"), (dict(table=0), "null"), (dict(blocks=0), "empty cache"),
    (dict(query=P + 8), "16 bytes"), (dict(keys=P + 2), "16 bytes"), (dict(values=P + 4), "16 bytes"),
    (dict(q_stride_head=68), "16 bytes"), (dict(kv_stride_pos=129), "16 bytes"),
    (dict(kv_stride_head=66), "16 bytes"), (dict(rows=1 << 30, tokens=1 << 30), "2\\^31"),
])
def test_attention_arguments(over, match):
    a = attention(**over)
    with pytest.raises(ValueError, match=match):
        ekv_hip.call("ekv_prefix_attention", ctypes.addressof(a), P, 1 << 40, 0)


def test_attention_workspace():
    a = attention()
    need = ekv_hip.load().ekv_prefix_attention_workspace(ctypes.addressof(a))
    assert need > 0
    for pointer, size in ((P, need - 1), (0, need), (P + 8, need)):
        with pytest.raises(ValueError, match="workspace"):
            ekv_hip.call("ekv_prefix_attention", ctypes.addressof(a), pointer, size, 0)
    assert ekv_hip.load().ekv_prefix_attention_workspace(ctypes.addressof(attention(head_dim=80))) == 0
    assert ekv_hip.load().ekv_prefix_attention_workspace(0) == 0


def test_attention_of_nothing_launches_nothing():
    a = attention(rows=0, tokens=0, query=0, out=0, lse=0)
    ekv_hip.call("ekv_prefix_attention", ctypes.addressof(a), 0, 0, 0)


def eviction(**over):
    a = ekv_hip.Eviction()
    base = dict(keys=P, values=P, kv_stride_block=4096, kv_stride_pos=128, kv_stride_head=64, blocks=10, table=P,
                table_stride=4, lens=P, seen=P, scores=P, positions=P, new_scores=P, new_positions=P, new_lens=2 * P,
                kv_dtype=ekv_hip.BF16, rows=3, kv_heads=2, head_dim=64, width=4, block_size=16, fixed_budget=8)
    for key, value in {**base, **over}.items():
        setattr(a, key, value)
    return a


@pytest.mark.parametrize("over,match", [
    (dict(kv_dtype=ekv_hip.F64), "type"), (dict(head_dim=80), "head dim"), (dict(rows=-1), "rows"),
    (dict(kv_heads=0), "heads"), (dict(block_size=0), "block size"), (dict(fixed_budget=-1), "budget"),
    (dict(recent=-1), "recent"), (dict(sinks=-1), "sinks"), (dict(width=1 << 27), "2\\^31"),
    (dict(rows=1 << 23), "rows"), (dict(lens=0), "null"), (dict(scores=0), "null"), (dict(seen=0), "null"),
    (dict(new_positions=0), "null"), (dict(new_lens=P), "lengths"), (dict(table_stride=3), "stride"),
    (dict(keys=P + 8), "16 bytes"), (dict(kv_stride_pos=130), "16 bytes"),
])
def test_eviction_arguments(over, match):
    a = eviction(**over)
    with pytest.raises(ValueError, match=match):
        ekv_hip.call("ekv_evict_tokens", ctypes.addressof(a), P, 1 << 40, 0)


def test_eviction_workspace():
    a = eviction()
    need = ekv_hip.load().ekv_evict_tokens_workspace(3, 2, 64)
    with pytest.raises(ValueError, match="workspace"):
        ekv_hip.call("ekv_evict_tokens", ctypes.addressof(a), P, need - 1, 0)
    assert ekv_hip.load().ekv_evict_tokens_workspace(-1, 2, 64) == 0


def test_python_checks_come_before_the_device():
    cache = torch.zeros(4, 2, 16, 2, 64, dtype=torch.bfloat16)
    query = torch.zeros(1, 8, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)

    def attend(match, **over):
        args = {**dict(query=query, kv_cache=cache, table=table, lens=lens, scale=0.1), **over}
        with pytest.raises(ValueError, match=match):
            prefix_attention(**args)

    attend("device tensor")
    attend("kv_cache", kv_cache=cache[0])
    attend("kv_cache", kv_cache=cache[:, :1])
    attend("contiguous rows", kv_cache=cache.transpose(3, 4).contiguous().transpose(3, 4))
    attend("query", query=query[0])
    attend("query", query=query[..., :32])
    attend("query", query=query.double())
    attend("table", table=table[0])
    attend("table", table=table.long())
    attend("lens", lens=lens.repeat(2))
    attend("q_start", q_start=lens)
    attend("prefix_lens", prefix_table=table)
    attend("prefix_table", prefix_lens=lens)
    attend("prefix_rows", prefix_table=table.repeat(2, 1), prefix_lens=lens.repeat(2))
    attend("prefix_lens", prefix_table=table, prefix_lens=lens.long())
    attend("out", out=query.float())
    attend("lse", lse=torch.zeros(1, 7))

    scores = torch.zeros(1, 2, 32)

    def evict(match, **over):
        args = {**dict(kv_cache=cache, table=table, lens=lens, scores=scores, positions=scores.int(), budget=4,
                       seen=lens), **over}
        with pytest.raises(ValueError, match=match):
            evict_tokens(**args)

    evict("device tensor")
    evict("kv_cache", kv_cache=cache[0])
    evict("scores", scores=scores[:, :, :31])
    evict("scores", scores=scores.double())
    evict("positions", positions=scores)
    evict("budget", budget=lens.long())
    evict("seen", seen=lens.repeat(2))
    evict("new_scores", new_scores=scores[0])


def test_attention_tables_of_the_most_keys():
    a = attention(width=(2**31 - 4096) // 16, block_size=16, table_stride=1 << 28)
    with pytest.raises(ValueError, match="2\\^31"):
        ekv_hip.call("ekv_prefix_attention", ctypes.addressof(a), P, 1 << 40, 0)
    a = attention(width=(2**31 - 4096) // 16 - 1, block_size=16, table_stride=1 << 28)
    with pytest.raises(ValueError, match="workspace"):
        ekv_hip.call("ekv_prefix_attention", ctypes.addressof(a), P, 0, 0)


def test_argument_blocks_are_the_structures():
    for kind in (ekv_hip.Attention, ekv_hip.Eviction):
        values = [i + 1 for i in range(len(kind._fields_))]
        block = kind.from_buffer_copy(ekv_hip.packer(kind)(*values))
        assert [getattr(block, name) for name, _ in kind._fields_] == values
    with pytest.raises(ValueError, match="range"):
        ekv_hip.packer(ekv_hip.Eviction)(*[2**40] * len(ekv_hip.Eviction._fields_))
