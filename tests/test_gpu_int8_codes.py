"""int8.Linear.codes where long rows are cut into parts of K: int32 sums in scratch, added
by a launch of their own.  Sums of codes are exact and the scales' products are the same,
so that codes(a, s) has the bits of the call on x = a s, and of one whole sum."""
import pytest
import torch

from ubridge_amd import int8, ops

pytestmark = pytest.mark.gpu

SIZES = [(1, 14336, 512), (16, 4096, 4096), (8, 8192, 1000), (40, 8192, 300), (16, 8190, 300), (64, 16384, 450), (33, 5000, 257)]


def make(dev, M, K, N, seed=0):
    g = torch.Generator().manual_seed(seed + M + K + N)
    a = torch.randint(-126, 127, (M, K), generator=g, dtype=torch.int8)
    a[:, K // 2] = 127  # every row's largest: x = a s is rounded to these codes
    s = torch.exp2(torch.randint(-6, 3, (M,), generator=g).float())
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8).to(dev)
    lin = int8.Linear(w, (torch.rand(N, generator=g) + 0.5).to(dev) / 100, torch.randn(N, generator=g).to(dev))
    return a.to(dev), s.to(dev), lin, w


@pytest.mark.parametrize("M,K,N", SIZES)
def test_values(dev, M, K, N):
    a, s, lin, w = make(dev, M, K, N)
    x = a.float() * s[:, None]
    sums = torch.round(a.double() @ w.t().double().contiguous())  # (below 2^53: exact)
    want = sums * s.double()[:, None] * lin.w_scale.double() + lin.bias.double()
    size = (sums * s.double()[:, None] * lin.w_scale.double()).abs() + lin.bias.double().abs()
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        got = lin.codes(a, s, dtype)
        # the sum to f32, two scales, the bias: four roundings, then the type's
        half = torch.finfo(dtype).eps / 2
        fits = want.abs() < torch.finfo(dtype).max
        assert bool(((got.double() - want).abs() <= half * want.abs() + 4 * 2.0**-24 * (1 + half) * size + 1e-30)[fits].all())
        if dtype == torch.float32:
            assert torch.equal(got, lin(x))
        guard = torch.full((M + 1, N), 3.0, device=dev, dtype=dtype)
        assert torch.equal(lin.codes(a, s, dtype, out=guard[:M]), got) and bool((guard[M] == 3.0).all())


@pytest.mark.parametrize("M,K,N", SIZES)
def test_caller_allocator(dev, M, K, N):
    # its scratch is the parts' sums alone: one block a call, so these sizes have parts
    a, s, lin, w = make(dev, M, K, N)
    want = lin.codes(a, s)
    alloc = ops.TorchWorkspaceAllocator()
    ops.set_workspace_allocator(alloc)
    try:
        got = lin.codes(a, s)
        torch.cuda.synchronize()
    finally:
        ops.set_workspace_allocator(None)
    assert alloc.calls == 1 and not alloc.live and torch.equal(got, want)


def test_graphs_of_one_stream_side_by_side(dev):
    # each has its own parts' sums: replayed at once on two streams, beside eager calls
    cases = [make(dev, 16, 4096, 4096, seed) for seed in (1, 2, 3)]
    want = [lin.codes(a, s).clone() for a, s, lin, w in cases]
    capture = torch.cuda.Stream()
    ops.release_workspace(capture)
    live = ops.workspace_stats()[0]
    graphs, outs = [], []
    for a, s, lin, w in cases[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=capture):
            outs.append(lin.codes(a, s))
        graphs.append(graph)
    assert ops.workspace_stats()[0] == live + 2
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(capture):
            a, s, lin, w = cases[2]
            got = lin.codes(a, s)
        torch.cuda.synchronize()
        assert all(torch.equal(o, t) for o, t in zip([*outs, got], want))
    del graphs, graph, outs
    ops.release_workspace(capture)
    assert ops.workspace_stats()[0] == live
