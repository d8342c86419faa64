"""Calls without a workspace inside graph captures: graphs replayed beside each other, beside eager
calls and after each other's end give what the calls give by themselves."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def pointers(monkeypatch):
    """The workspace addresses of the calls from now on."""
    from dels_b200 import _lib

    seen = []
    call = _lib.call

    def spy(name, *args):
        at = {"dels_beam_select": 17, "dels_linear_w8a8": 13, "dels_linear_bf16": 10}.get(name)
        if at is not None:
            seen.append(getattr(args[at], "value", None))
        return call(name, *args)

    monkeypatch.setattr(_lib, "call", spy)
    return seen


def capture(call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


def operators(dev):
    from dels_b200 import ops

    g = torch.Generator(device=dev).manual_seed(4)
    wq, sw = ops.quantize_rows_i8(torch.randn(2000, 512, generator=g, device=dev))
    w = torch.randn(512, 512, generator=g, device=dev).bfloat16()

    def select(rows, V):
        x = torch.randn(rows, V, generator=g, device=dev)
        s = torch.zeros(rows // 4, 4, device=dev)
        return lambda: torch.cat([t.flatten().double() for t in vars(ops.beam_select(x, s)).values()])

    def product(rows):
        x = torch.randn(rows, 512, generator=g, device=dev).bfloat16()
        return lambda: ops.linear_w8a8(x, wq, sw)

    def linear(rows):
        x = torch.randn(rows, 512, generator=g, device=dev).bfloat16()
        return lambda: ops.linear_bf16(x, w)

    return {"select": (select(64, 20000), select(64, 20000), select(2048, 40000)),
            "product": (product(40), product(40), product(4000)), "linear": (linear(40), linear(40), linear(4000))}


@pytest.mark.parametrize("name", ["select", "product", "linear"])
def test_graphs_beside_each_other(cuda_device, monkeypatch, name):
    one, two, large = operators(cuda_device)[name]
    want = [one().clone(), two().clone()]
    seen = pointers(monkeypatch)
    eager = one()
    graphs = [capture(one), capture(two)]
    assert len(seen) == 3 and len(set(seen)) == 3 and None not in seen
    large()  # needs a larger workspace than any before
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(50):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        large()
    torch.cuda.synchronize()
    assert torch.equal(eager, want[0])
    for (_, out), w in zip(graphs, want):
        assert torch.equal(out, w)
    # the first graph's end leaves the second one its workspace
    graph, out = graphs.pop()
    graphs[0][0].reset()
    del graphs
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want[1])


def test_calls_of_one_capture_share_a_workspace(cuda_device, monkeypatch):
    one, two, _ = operators(cuda_device)["product"]
    want = [one().clone(), two().clone()]
    seen = pointers(monkeypatch)
    graph, outs = capture(lambda: [one(), two()])
    assert len(set(seen)) == 1
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
