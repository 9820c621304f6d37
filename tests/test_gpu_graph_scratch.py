"""Scratch of captured graphs: a program that captures again and again, destroying what it
captured before, holds no more of it than one that captures once or twice."""
import gc

import pytest
import torch

from ubridge_amd import moe, mx, norm, ops

pytestmark = pytest.mark.gpu


def test_capture_destroy_capture(dev):
    g = torch.Generator().manual_seed(0)
    lin = mx.Linear(*mx.quantize(torch.randn(200, 2000, generator=g).to(dev)), 2000)
    experts = [torch.randn(*s, generator=g).bfloat16().to(dev) / 16 for s in ((8, 64, 256), (8, 256, 32))]
    layer = moe.FusedMoE(*experts, topk=2)
    n = norm.RmsNorm(torch.rand(2000, generator=g).to(dev).requires_grad_())

    def run(big, dy, x, lg):
        return [lin(big), layer.decode(x, lg), torch.autograd.grad(n(big), [n.weight], dy)[0]]
    ins = [[torch.randn(m, c, generator=g).bfloat16().to(dev) for m, c in ((rows, 2000), (rows, 2000), (12, 256), (12, 8))]
           for rows in (300, 40)]
    want = [[t.clone() for t in run(*i)] for i in ins]
    stream = torch.cuda.Stream()
    ops.release_workspace(stream)
    before = ops.workspace_stats()[:2]
    seen = []
    for turn in range(12):
        i = turn % 2
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = run(*ins[i])
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i])), turn
        seen.append(ops.workspace_stats()[0] - before[0])
        del graph, out
        gc.collect()
        torch.cuda.synchronize()
    # (the runtime may tell of a graph's end some graphs later; of all twelve it would be 12)
    assert max(seen) <= 6 * seen[0], seen
    # two that live side by side keep what is theirs
    graphs, outs = [], []
    for i in ins:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(run(*i))
        graphs.append(graph)
    for _ in range(3):
        for graph, out, w in zip(graphs, outs, want):
            graph.replay()
            with torch.cuda.stream(stream):
                run(*ins[0])
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w))
    del graphs, graph, outs, out
    gc.collect()
    ops.release_workspace(stream)
    assert ops.workspace_stats()[:2] == before
