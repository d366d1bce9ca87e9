"""The workspace of a captured int8_linear is the graph's own memory: calls outside it, and other graphs, are never given it."""
import pytest
import torch

import gonngpu as G
from tests import int8_ref as R
from tests.test_int8_gpu import _ints, _stored, _x

pytestmark = pytest.mark.gpu


def test_workspace_of_a_captured_call(dev, monkeypatch):
    M, N, K = 300, 200, 5000
    x, b = _x(M, K, torch.float16, 1), _ints(N, K, 2)
    xd, bd, y = x.to(dev), _stored(dev, b), torch.empty((M, N), device=dev)
    G.int8_linear(xd, (bd, None), y)
    torch.cuda.synchronize()
    taken, alloc = [], G._alloc
    monkeypatch.setattr(G, "_alloc", lambda n, s: taken.append(alloc(n, s)) or taken[-1])
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph in graphs:
        with torch.cuda.graph(graph):
            G.int8_linear(xd, (bd, None), y)
    assert len(taken) == 2 and taken[0] != taken[1]
    for graph, at in zip(graphs, taken):
        own = [s for s in torch.cuda.memory_snapshot() if s["address"] <= at < s["address"] + s["total_size"]]
        assert len(own) == 1 and tuple(own[0]["segment_pool_id"]) == tuple(graph.pool())
    # Nothing else is given that memory while the graphs are there, and what others write does not reach their results.
    others = [torch.full((M * K // 4,), 1e30, device=dev) for _ in range(40)]
    want = R.product(*R.quantize(x), b, None)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for graph, s in zip(graphs, streams):  # together
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y.cpu(), want) and all(bool((o == 1e30).all()) for o in others)
