"""Scratch of the 8-bit cache's attention: ticket rows of captured calls."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
pkg = importlib.import_module("numerics-and-sparse-attn_b200")
KV8 = importlib.import_module("numerics-and-sparse-attn_b200.kv8")


def test_more_captured_calls_than_ticket_rows(monkeypatch):
    """With three rows for 3 x 4 captured calls: no graph is given what another holds, and graphs replayed side by side,
    again and again, give the eager calls' bits and leave the tickets zero."""
    hkv, group, d, n = 2, 8, 64, 6000
    g = torch.Generator(device=DEV).manual_seed(60)
    caches = [pkg.Kv8Cache(2, hkv, n, head_dim=d, device=DEV) for _ in range(3)]
    for c in caches:
        c.append(*(torch.randn(2, hkv, n, d, device=DEV, generator=g).half() for _ in range(2)))
    qs = [torch.randn(2, hkv * group, d, device=DEV, generator=g).half() for _ in range(3)]
    want = [c.attend(q) for c, q in zip(caches, qs)]
    index = torch.cuda.current_device()
    rows = torch.zeros_like(KV8._graph[index][0][:3])
    monkeypatch.setattr(KV8, "_GRAPH_ROWS", 3)
    monkeypatch.setitem(KV8._graph, index, [rows, 0])
    given, real = [], KV8._scratch

    def spy(*args):
        pair = real(*args)
        given[-1].append(pair[1].data_ptr())
        return pair

    monkeypatch.setattr(KV8, "_scratch", spy)
    graphs, outs = [], []
    for c, q in zip(caches, qs):
        graph = torch.cuda.CUDAGraph()
        given.append([])
        with torch.cuda.graph(graph):
            outs.append([c.attend(q) for _ in range(4)])
        graphs.append(graph)
    assert all(len(x) == 4 for x in given)
    assert not any(set(given[i]) & set(given[j]) for i in range(3) for j in range(i))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(3) for o in outs[i])
    assert not rows.any() and pkg.device_error(torch.device(DEV)) == 0
