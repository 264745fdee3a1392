"""Graphs of layers with the default workspace, next to each other and to eager calls."""
import pytest
import torch

from tests._helpers import banner
from tests.test_gpu_threads import _int4, _mxfp4, _routed

pytestmark = pytest.mark.gpu

KINDS = pytest.mark.parametrize("make", [_int4, _mxfp4, _routed], ids=["int4", "mxfp4", "routed"])


def _captured(call, stream):
    with torch.cuda.stream(stream):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = call()
    return graph, out


@KINDS
@pytest.mark.parametrize("T", [16, 48, 300])
def test_two_graphs_at_once(make, T, device):
    """Captured on one stream one after the other, replayed on two."""
    banner(f"two graphs {make.__name__} T={T}")
    calls = [make(T, 5, device), make(T, 6, device)]
    want = [call() for call in calls]
    stream = torch.cuda.Stream()
    pairs = [_captured(call, stream) for call in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _, out in pairs:
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for (graph, _), s in zip(pairs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (_, out), ref in zip(pairs, want):
        assert torch.equal(out, ref)


@KINDS
def test_replays_touch_nothing_after_a_larger_call(make, device):
    """The stream's workspace grows after the capture; what takes the memory that it lets go
    of is not written by the replays."""
    banner(f"graph and a larger call {make.__name__}")
    small, large = make(16, 5, device), make(2000, 6, device)
    want, stream = small(), torch.cuda.Stream()
    graph, out = _captured(small, stream)
    with torch.cuda.stream(stream):
        large()
        others = [torch.full((1 << 20,), 7, dtype=torch.uint8, device=device) for _ in range(64)]
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(bool((t == 7).all()) for t in others)
