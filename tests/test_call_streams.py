"""A call with ``stream=`` allocates on that stream: what torch hands out and takes back is ordered by the stream that was
current when it was allocated, so a workspace or an output from any other one is shared with that one's other work.

On the host, with the library replaced by one that launches nothing: every torch operation that a call makes is noted with
the stream that was current then."""

import types

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import ekv_hip
import observe.allocation
import observe.controller
import observe.tile_shares
import runtime.eviction
import runtime.prefix_attention

SIDE = types.SimpleNamespace(cuda_stream=77)


class Noted(TorchDispatchMode):
    """(operation, current stream) of the operations that give new tensors."""

    def __init__(self, current):
        super().__init__()
        self.current, self.made = current, []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        result = func(*args, **(kwargs or {}))
        if isinstance(result, torch.Tensor) and func.overloadpacket not in (torch.ops.aten.detach, torch.ops.aten.view):
            self.made.append((str(func), self.current[-1]))
        return result


@pytest.fixture
def host(monkeypatch):
    """A library that notes (entry point, stream) of each launch, torch's current stream, and checks that let host
    tensors pass."""
    current, launches = [None], []

    class Context:
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            current.append(self.stream)

        def __exit__(self, *_):
            current.pop()

    class Library:
        def __getattr__(self, name):
            if name.endswith("_workspace") or name.endswith("_bytes"):
                return lambda *args: 64

            def launch(*args):
                launches.append((name, args[-1]))
                return 0

            return launch

    monkeypatch.setattr(torch.cuda, "stream", Context)
    monkeypatch.setattr(ekv_hip, "_lib", Library())
    monkeypatch.setattr(ekv_hip, "stream_handle", lambda stream=None: (stream or current[-1]).cuda_stream)
    return types.SimpleNamespace(current=current, launches=launches, patch=monkeypatch)


def check(host, module, call, least):
    host.patch.setattr(module, "check_tensors", lambda *specs: torch.device("cpu"))
    with Noted(host.current) as noted:
        call()
    assert len(noted.made) >= least
    assert all(stream is SIDE for _, stream in noted.made), noted.made
    assert host.launches and all(stream == 77 for _, stream in host.launches)


def cache_and_rows():
    rows = torch.zeros(3, dtype=torch.int32)
    return torch.zeros(4, 2, 16, 2, 64, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32), rows


def test_attention(host):
    cache, table, lens = cache_and_rows()
    query = torch.zeros(3, 8, 64, dtype=torch.bfloat16)
    check(host, runtime.prefix_attention, lambda: runtime.prefix_attention.prefix_attention(
        query, cache, table, lens, 0.1, stream=SIDE), 3)


def test_eviction(host):
    cache, table, lens = cache_and_rows()
    scores, positions = torch.zeros(3, 2, 32), torch.zeros(3, 2, 32, dtype=torch.int32)
    check(host, runtime.eviction, lambda: runtime.eviction.evict_tokens(
        cache, table, lens, scores, positions, 4, lens, stream=SIDE), 4)


@pytest.mark.parametrize("objective", ["maxmin", "sum"])
def test_objectives(host, objective):
    scores, blocks = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int32)
    keep = observe.allocation.maxmin_keep if objective == "maxmin" else observe.allocation.sum_keep
    check(host, observe.allocation, lambda: keep(scores, blocks, budget=2, stream=SIDE), 4)  # with the float64 scores


def test_uniform(host):
    scores, blocks = torch.zeros(3, 8, dtype=torch.float64), torch.zeros(3, dtype=torch.int32)
    check(host, observe.allocation, lambda: observe.allocation.uniform_keep(scores, blocks, stream=SIDE), 3)


@pytest.mark.parametrize("objective", ["uniform", "maxmin", "sum"])
def test_controller(host, objective):
    shares, lengths, evidence = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int32), torch.ones(3, dtype=torch.bool)
    host.patch.setattr(observe.allocation, "check_tensors", lambda *specs: torch.device("cpu"))
    check(host, observe.controller, lambda: observe.controller.keep_rows(
        shares, lengths, evidence, 0.5, objective=objective, stream=SIDE), 2)


def test_shares(host):
    host.patch.setattr(torch.Tensor, "is_cuda", True)
    out = torch.zeros(3, 8)
    check(host, observe.allocation, lambda: observe.tile_shares.tile_shares(
        4096, table_layers=2, layers=2, rows=3, width=8, group_rows=4, row_ids=None, row_blocks=None, tile_blocks=8,
        out=out, stream=SIDE), 1)


def test_raw_handles(monkeypatch):
    device = torch.device("cuda:0")
    tensor = types.SimpleNamespace(device=device)
    monkeypatch.setattr(torch.cuda, "stream", lambda stream: ("under", stream))
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, device: (handle, device))
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device: ("default", device))
    assert ekv_hip.on_stream(SIDE, tensor) == ("under", SIDE)
    assert ekv_hip.on_stream(4096, tensor) == ("under", (4096, device))
    assert ekv_hip.on_stream(0, tensor) == ("under", ("default", device))  # 0 is the default stream's handle
    assert ekv_hip.on_stream(4096, device) == ("under", (4096, device))
    with ekv_hip.on_stream(None, tensor), ekv_hip.on_stream(4096, torch.zeros(1)):
        pass  # no stream named; a host tensor, which the call's checks refuse


@pytest.mark.gpu
def test_two_streams_beside_other_work():
    """Two calls on streams of their own, with the current stream's tensors made and dropped around them."""
    from attention_cases import Batch, check as within

    batches = [Batch([700, 300, 90], prefixes=[70], seed=s).with_scores() for s in (31, 32)]
    inputs = [b.on_gpu() for b in batches]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    wants = [b.want() for b in batches]
    torch.cuda.synchronize()
    results = []
    for args, stream in zip(inputs, streams):
        results.append(runtime.prefix_attention.prefix_attention(
            **args, stream=stream if stream is streams[0] else stream.cuda_stream))
        for size in (1 << 10, 1 << 16, 1 << 22):
            torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for b, args, want, (out, lse) in zip(batches, inputs, wants, results):
        within(b, out, lse, args["scores"], want)
