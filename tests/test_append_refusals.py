"""What appending tokens and rotating heads refuse, on the host: the C ABI's checks (which need no GPU) and the Python
layer's; the sections of several axes; and the device and stream a call runs on."""

import ctypes
import types

import pytest
import torch

import ekv_hip
import runtime.append
import runtime.rotary
from runtime.append import append_tokens
from runtime.rotary import rotary_frequencies, rotate_heads, section_axes

P = 4096  # a placeholder device address: the checks refuse the call before using it


def block(kind, base, over):
    a = kind()
    for key, value in {**base, **over}.items():
        setattr(a, key, value)
    return a


def rotation(**over):
    return block(ekv_hip.Rotation, dict(
        query=P, q_stride_token=512, q_stride_head=64, key=P, k_stride_token=128, k_stride_head=64, q_out=P,
        q_out_stride_token=512, q_out_stride_head=64, k_out=P, k_out_stride_token=128, k_out_stride_head=64, positions=P,
        frequencies=P, dtype=ekv_hip.BF16, weight_dtype=ekv_hip.BF16, tokens=3, q_heads=8, kv_heads=2, head_dim=64, pairs=32,
        axis_count=1, rotary_scale=1.0, eps=1e-6), over)


@pytest.mark.parametrize("over,match", [
    (dict(dtype=ekv_hip.FP8_E4M3), "type"), (dict(dtype=ekv_hip.F64), "type"), (dict(q_weight=P, weight_dtype=ekv_hip.F16), "type"),
    (dict(head_dim=8), "head dim"), (dict(head_dim=72), "head dim"), (dict(head_dim=272), "head dim"), (dict(pairs=-8), "pairs"),
    (dict(pairs=12), "pairs"), (dict(pairs=40), "pairs"), (dict(tokens=-1), "tokens"), (dict(q_heads=-1), "heads"),
    (dict(kv_heads=(1 << 20) + 1), "heads"), (dict(frequencies=0), "null"), (dict(positions=0), "null"), (dict(query=0), "null"),
    (dict(q_out=0), "null"), (dict(key=0), "null"), (dict(k_out=0), "null"), (dict(axis_count=0), "axes"),
    (dict(axis_count=2, positions_stride=-1), "axes"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(query=P + 8), "16 bytes"), (dict(k_out=P + 2), "16 bytes"), (dict(q_stride_head=68), "16 bytes"),
    (dict(k_stride_token=129), "16 bytes"), (dict(q_out_stride_token=4), "16 bytes"), (dict(q_weight=P + 4), "16 bytes"),
    (dict(k_weight=P, k_weight_stride=20), "16 bytes"), (dict(tokens=(1 << 26) - 64), "launch"),
])
def test_rotation_arguments(over, match):
    a = rotation(**over)
    with pytest.raises(ValueError, match=match):
        ekv_hip.call("ekv_rotate_heads", ctypes.addressof(a), 0)


def appending(**over):
    return block(ekv_hip.Append, dict(
        query=P, q_stride_token=512, q_stride_head=64, new_keys=P, new_values=P, k_stride_token=128, k_stride_head=64,
        v_stride_token=128, v_stride_head=64, q_out=P, q_out_stride_token=512, q_out_stride_head=64, keys=P, values=P,
        kv_stride_block=4096, kv_stride_pos=128, kv_stride_head=64, blocks=10, table=P, table_stride=4, lens=P,
        frequencies=P, dtype=ekv_hip.BF16, weight_dtype=ekv_hip.BF16, kv_dtype=ekv_hip.BF16, rows=3, width=4, tokens=3,
        max_query=1, q_heads=8, kv_heads=2, head_dim=64, block_size=16, pairs=32, axis_count=1, rotary_scale=1.0, eps=1e-6,
        k_scale=1.0, v_scale=1.0), over)


@pytest.mark.parametrize("over,match", [
    (dict(dtype=ekv_hip.FP8_E4M3, kv_dtype=ekv_hip.FP8_E4M3), "type"), (dict(kv_dtype=ekv_hip.F16), "type"),
    (dict(kv_dtype=ekv_hip.F64), "type"), (dict(head_dim=40), "head dim"), (dict(head_dim=0), "head dim"),
    (dict(pairs=36), "pairs"), (dict(rows=-1), "rows"), (dict(width=-1), "width"), (dict(blocks=-1), "rows"),
    (dict(max_query=0), "tokens a row"), (dict(kv_heads=0), "heads"), (dict(block_size=0), "block size"),
    (dict(tokens=4), "q_start"), (dict(max_query=2), "q_start"), (dict(width=1 << 27, table_stride=1 << 28), "2\\^31"),
    (dict(k_scale=0.0), "scales"), (dict(v_scale=-1.0), "scales"), (dict(k_scale=float("nan")), "scales"),
    (dict(rows=0, q_start=P), "no row"), (dict(new_keys=0), "null"), (dict(new_values=0), "null"), (dict(lens=0), "null"),
    (dict(query=0), "null"), (dict(q_out=0), "null"), (dict(keys=0), "null"), (dict(values=0), "null"), (dict(table=0), "null"),
    (dict(blocks=0), "empty cache"), (dict(new_keys=P + 8), "16 bytes"), (dict(new_values=P + 2), "16 bytes"),
    (dict(keys=P + 4), "16 bytes"), (dict(values=P + 8), "16 bytes"), (dict(kv_stride_pos=129), "16 bytes"),
    (dict(kv_stride_head=68), "16 bytes"), (dict(kv_stride_block=4097), "16 bytes"), (dict(v_stride_head=4), "16 bytes"),
    (dict(k_weight=P + 8), "16 bytes"), (dict(table_stride=3), "stride"), (dict(rows=1 << 26, tokens=(1 << 26)), "launch"),
    (dict(positions=P, axis_count=0), "axes"), (dict(eps=-1.0), "eps"), (dict(tokens=-1), "tokens"),
])
def test_append_arguments(over, match):
    a = appending(**over)
    with pytest.raises(ValueError, match=match):
        ekv_hip.call("ekv_append_tokens", ctypes.addressof(a), 0)


def test_nothing_launches_nothing():
    for name, a in (("ekv_rotate_heads", rotation(tokens=0, query=0)), ("ekv_rotate_heads", rotation(q_heads=0, kv_heads=0)),
                    ("ekv_append_tokens", appending(rows=0, tokens=0, new_keys=0)),
                    ("ekv_append_tokens", appending(tokens=0, q_start=P, lens=0))):
        ekv_hip.call(name, ctypes.addressof(a), 0)
    for name in ("ekv_rotate_heads", "ekv_append_tokens"):
        with pytest.raises(ValueError, match="null"):
            ekv_hip.call(name, 0, 0)


def test_argument_blocks_are_the_structures():
    for kind in (ekv_hip.Rotation, ekv_hip.Append):
        values = [i + 1 for i in range(len(kind._fields_))]
        packed = kind.from_buffer_copy(ekv_hip.packer(kind)(*values))
        assert [getattr(packed, name) for name, _ in kind._fields_] == values


def test_python_checks_come_before_the_device():
    query, key = torch.zeros(3, 8, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    at, turning = torch.zeros(3, dtype=torch.int32), torch.ones(32, dtype=torch.float64)

    def rotate(match, **over):
        args = {**dict(query=query, key=key, positions=at, frequencies=turning), **over}
        with pytest.raises(ValueError, match=match):
            rotate_heads(**args)

    rotate("device tensor")
    rotate("query", query=query[0])
    rotate("query", query=query.double())
    rotate("key", key=key[:2])
    rotate("key", key=key.float())
    rotate("key", key=key[..., :32])
    rotate("k_out", key=None, k_out=key)
    rotate("k_weight", key=None, k_weight=torch.ones(64))
    rotate("positions", positions=None)
    rotate("contiguous rows", query=query.transpose(1, 2).contiguous().transpose(1, 2))
    rotate("q_out", q_out=query[:2])
    rotate("k_out", k_out=key.float())

    cache = torch.zeros(4, 2, 16, 2, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)

    def append(match, **over):
        args = {**dict(kv_cache=cache, table=table, lens=lens, keys=key, values=key, query=query, frequencies=turning), **over}
        with pytest.raises(ValueError, match=match):
            append_tokens(**args)

    append("device tensor")
    append("kv_cache", kv_cache=cache[0])
    append("cache", kv_cache=cache.half())
    append("table", table=table[0])
    append("table", table=table.long())
    append("lens", lens=lens[:2])
    append("keys", keys=key[:, :1])
    append("keys", keys=key[..., :32])
    append("values", values=key[:2])
    append("values", values=key.float())
    append("values", keys=key[:0], values=key, query=None)
    append("query", query=query[:2])
    append("query", query=query.float())
    append("need a query", query=None, q_out=query)
    append("need a query", query=None, q_weight=torch.ones(64))
    append("q_start", q_start=lens)
    append("seen", seen=lens.long())
    append("need frequencies", frequencies=None, positions=at)


@pytest.fixture
def host(monkeypatch):
    """A library that notes (entry point, arguments, stream), and checks that let host tensors pass."""
    launches = []
    monkeypatch.setattr(ekv_hip, "_raw_stream", None)

    class Library:
        def __getattr__(self, name):
            def launch(arguments, stream):
                launches.append((name, arguments, stream))
                return 0

            return launch

    monkeypatch.setattr(ekv_hip, "_lib", Library())
    monkeypatch.setattr(ekv_hip, "stream_handle", lambda stream=None: 5 if stream is None else stream.cuda_stream)
    for module in (runtime.append, runtime.rotary):
        monkeypatch.setattr(module, "check_tensors", lambda *specs: types.SimpleNamespace(index=-1))
    return types.SimpleNamespace(launches=launches, patch=monkeypatch)


def test_rotary_and_weights_are_checked(host):
    x, at = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32)
    turning = torch.ones(32, dtype=torch.float64)

    def refused(match, positions=at, frequencies=turning, **over):
        with pytest.raises(ValueError, match=match):
            rotate_heads(x, x, positions, frequencies, **over)

    refused("frequencies", frequencies=torch.ones(2, 16))
    refused("pairs", frequencies=torch.ones(33, dtype=torch.float64))
    refused("positions", positions=at[:2])
    refused("positions", positions=at.view(1, 1, 3))
    refused("need axes", positions=at.expand(2, 3))
    refused("need frequencies", positions=None, frequencies=None, axes=at)
    refused("q_weight", q_weight=torch.ones(32))
    refused("q_weight", q_weight=torch.ones(3, 64))
    refused("k_weight", k_weight=torch.ones(64, dtype=torch.float16))
    assert not host.launches
    half = x.half()
    with pytest.raises(ValueError, match="as q_weight"):
        rotate_heads(half, half, at, turning, q_weight=torch.ones(64), k_weight=torch.ones(64).half())
    cache, table = torch.zeros(4, 2, 16, 2, 64), torch.zeros(3, 2, dtype=torch.int32)
    lens = torch.ones(3, dtype=torch.int32)

    def refused_append(match, **over):
        with pytest.raises(ValueError, match=match):
            append_tokens(**{**dict(kv_cache=cache, table=table, lens=lens, keys=x, values=x, frequencies=turning), **over})

    refused_append("first", first=lens.long())
    refused_append("first", first=lens[:2])
    refused_append("scores", scores=torch.zeros(3, 2, 31))
    refused_append("slot_positions", slot_positions=torch.zeros(2, 2, 32, dtype=torch.int32))
    refused_append("axes need positions", axes=torch.zeros(32, dtype=torch.int32))
    refused_append("range", max_query=2**40)
    assert not host.launches


def test_what_is_passed(host):
    x, at = torch.zeros(3, 6, 64, dtype=torch.bfloat16), torch.arange(6, dtype=torch.int32).view(2, 3)
    turning, axes = torch.ones(16, dtype=torch.float64), torch.zeros(16, dtype=torch.int32)
    weight = torch.ones(2, 64)
    rotate_heads(x[:, :4], x[:, 4:], at, turning, axes=axes, adjacent=True, k_weight=weight, weight_offset=1.0)
    name, packed, stream = host.launches.pop()
    a = ekv_hip.Rotation.from_buffer_copy(packed)
    assert (name, stream) == ("ekv_rotate_heads", 5)
    assert (a.q_stride_token, a.q_stride_head, a.key - a.query, a.q_out_stride_token) == (384, 64, 512, 256)
    assert (a.positions, a.positions_stride, a.axis_count, a.axes, a.pairs, a.adjacent) == (at.data_ptr(), 3, 2, axes.data_ptr(), 16, 1)
    assert (a.q_weight, a.k_weight, a.k_weight_stride, a.weight_dtype) == (None, weight.data_ptr(), 64, ekv_hip.F32)
    cache, table = torch.zeros(4, 2, 16, 2, 64, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32)
    lens, prefix = torch.ones(3, dtype=torch.int32), torch.full((1,), 9, dtype=torch.int32)
    scores = torch.zeros(3, 2, 40)
    assert append_tokens(cache, table, lens, x[:, :2], x[:, 2:4], first=prefix.expand(3), scores=scores, advance=True) is None
    name, packed, stream = host.launches.pop()
    a = ekv_hip.Append.from_buffer_copy(packed)
    assert (name, stream, a.query, a.q_heads, a.pairs, a.saturate, a.advance) == ("ekv_append_tokens", 5, None, 0, 0, 1, 1)
    assert (a.first, a.first_stride, a.values - a.keys, a.scores_stride_row) == (prefix.data_ptr(), 0, 2 * 2048, 80)
    assert a.new_values - a.new_keys == 256 and a.blocks == 4 and a.table_stride == 2


def test_a_stream_is_what_a_call_allocates_on(host):
    """With ``stream=`` every output is made while that stream is the current one, and the launch goes to it."""
    current, made = [None], []

    class Context:
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            current.append(self.stream)

        def __exit__(self, *_):
            current.pop()

    empty = torch.empty

    def noted(*args, **kwargs):
        made.append(current[-1])
        return empty(*args, **kwargs)

    host.patch.setattr(torch.cuda, "stream", Context)
    host.patch.setattr(torch, "empty", noted)
    side = types.SimpleNamespace(cuda_stream=77)
    x = torch.zeros(3, 2, 64)
    rotate_heads(x, x, None, None, stream=side)
    cache, table = torch.zeros(4, 2, 16, 2, 64), torch.zeros(3, 2, dtype=torch.int32)
    append_tokens(cache, table, torch.ones(3, dtype=torch.int32), x, x, query=x, stream=side)
    assert made == [side] * 3 and [stream for _, _, stream in host.launches] == [77, 77]


def test_another_device_and_its_streams(monkeypatch):
    """A call on tensors of another device makes it the current one; a stream of a third is refused."""
    entered = []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            entered.append(self.index)

        def __exit__(self, *_):
            pass

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "stream", lambda stream: ("under", stream))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=0: types.SimpleNamespace(cuda_stream=100 + device))
    monkeypatch.setattr(ekv_hip, "stream_handle", lambda stream=None: 9 if stream is None else stream.cuda_stream)
    there = types.SimpleNamespace(get_device=lambda: 1, device=torch.device("cuda:1"))
    here = types.SimpleNamespace(get_device=lambda: 0, device=torch.device("cuda:0"))
    side = types.SimpleNamespace(cuda_stream=77, device=torch.device("cuda:0"))
    for raw in (None, (lambda device: 200 + device, lambda: 0)):  # before and after the first call
        monkeypatch.setattr(ekv_hip, "_raw_stream", raw)
        context, handle = ekv_hip.beside(None, there)
        with context:
            assert entered.pop() == 1 and handle == 101
        assert ekv_hip.beside(None, here) == (None, 9 if raw is None else 200)
        assert ekv_hip.beside(side, here) == (("under", side), 77)
        with pytest.raises(ValueError, match="stream"):
            ekv_hip.beside(side, there)
        assert ekv_hip.beside(None, torch.zeros(1)) == (None, 9)


def test_sections():
    def axes(*pairs, **over):
        return section_axes(*pairs, device="cpu", **over).tolist()

    assert axes(2, 1, 3) == [0, 0, 1, 2, 2, 2]
    assert axes(4) == [0, 0, 0, 0]
    assert axes(4, 2, 2, interleaved=True) == [0, 1, 2, 0, 1, 2, 0, 0]
    assert axes(3, 3, 2, interleaved=True) == [0, 1, 2, 0, 1, 2, 0, 1]
    assert axes(4, 0, 2, interleaved=True) == [0, 0, 2, 0, 0, 2]
    for bad in ((), (2, -1)):
        with pytest.raises(ValueError, match="sections"):
            axes(*bad)
    with pytest.raises(ValueError, match="fit"):
        axes(0, 3, 1, interleaved=True)
    f = rotary_frequencies(4, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    for bad in ((0, 10.0), (4, 0.0)):
        with pytest.raises(ValueError, match="pairs"):
            rotary_frequencies(*bad, device="cpu")


@pytest.mark.parametrize("over", [dict(seen=P), dict(seen=P + 8), dict(first=P + 4), dict(first=P - 16, first_stride=2), dict(seen=2 * P, first=2 * P)])
def test_counts_that_share_memory_do_not_advance(over):
    """lens and seen both grow by a row's tokens, while other rows' tokens may still read `first`."""
    a = appending(lens=P, advance=1, **over)
    with pytest.raises(ValueError, match="memory"):
        ekv_hip.call("ekv_append_tokens", ctypes.addressof(a), 0)


def test_first_of_a_negative_stride():
    with pytest.raises(ValueError, match="stride"):
        ekv_hip.call("ekv_append_tokens", ctypes.addressof(a := appending(first=2 * P, first_stride=-1)), 0)
