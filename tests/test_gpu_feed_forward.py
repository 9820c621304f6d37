"""The norm and the feed-forward operators together, as examples/feed_forward.py runs
them, against the same halves in 64 bits.

Tolerance, in norm per half: roundings of the normed values, gate and up, the gated
activations and the result to bf16 (2^-9 of a value, half a step, each at most 2^-8 in
norm), and where one moves a value across a border of its code, one code: of e4m3
blocks 2^-4 of those few values, of int8 one of 127.  A share of 2^-4 of all values
(what a bf16 step covers of a code's) moved by 2^-3 adds 2^-5 in norm at most, once for
each of the two roundings to blocks: 2 * 2^-5 + 4 * 2^-8 < 2^-3.
"""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT
from test_gpu_mx import blocks, values
from ubridge_amd import moe, mx, norm

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location("feed_forward", os.path.join(ROOT, "examples", "feed_forward.py"))
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)


def normed(n, h):
    d = h.double()
    return d / torch.sqrt((d * d).mean(1, keepdim=True) + n.eps) * n.weight.double()


def in_blocks(x, fmt):
    return values(*blocks(x, fmt), fmt)[:, :x.shape[1]].to(x.device)


def dense(n, h, w13, w2, act):
    g, u = (in_blocks(normed(n, h), act) @ in_blocks(w13, "fp4").t().contiguous()).chunk(2, 1)
    a = torch.nn.functional.silu(g) * u
    return in_blocks(a, act) @ in_blocks(w2, "fp4").t().contiguous()


def experts(n, h, half):
    y, layer = normed(n, h), half.layer
    lg = y @ half.router.double()
    out = torch.zeros_like(y)
    top = torch.topk(lg, layer.topk, 1)
    w = torch.softmax(top.values, 1)
    for t in range(len(y)):
        for e, p in zip(top.indices[t].tolist(), w[t]):
            w13 = layer.w13[e].double() * layer.s13[e].double()[:, None]
            w2 = layer.w2[e].double() * layer.s2[e].double()[:, None]
            g, u = (w13 @ y[t]).chunk(2)
            out[t] += p * (w2 @ (torch.nn.functional.silu(g) * u))
    return out


def near(got, want):
    assert float((got.double() - want).norm() / want.norm()) < 2.0**-3


@pytest.mark.parametrize("tokens", [1, 7, 16])
def test_halves(dev, tokens):
    g = torch.Generator().manual_seed(tokens)
    hidden, inner, E, k = 192, 96, 12, 3
    halves, head = example.build(2, hidden, inner, E, k, 40, g)
    w13, w2 = (torch.randn(*s, generator=g).bfloat16().to(dev) * s[-1] ** -0.5 for s in ((2 * inner, hidden), (hidden, inner)))
    n, ex = halves[1]
    for act in ("fp8", "fp4"):
        x, r = (torch.randn(tokens, hidden, generator=g).bfloat16().to(dev) for _ in "xr")
        h = (x.float() + r.float()).bfloat16()
        half = example.Dense(w13, w2, act)
        y, s = half(n, x, r)
        assert s.data_ptr() == r.data_ptr() and torch.equal(s, h)
        if act == "fp8":  # (steps of e2m1 are a quarter to a half of a value)
            near(y, dense(n, h, w13, w2, act))
        # the blocks that the norm made are those of its f32 result
        q = n(h, quant=act)
        near(half.w13.codes(*q, torch.float32), mx.dequantize(*q, hidden, torch.float32).double()
             @ in_blocks(w13, "fp4").t().contiguous())
    r = torch.randn(tokens, hidden, generator=g).bfloat16().to(dev)
    h = (x.float() + r.float()).bfloat16()
    y, s = ex(n, x, r)
    assert torch.equal(s, h)
    near(y, experts(n, h, ex))
    n, last = head
    lin = last.linear
    w = lin.w[:, :hidden].double() * lin.w_scale.double()[:, None]
    near(last(n, y, s), normed(n, (y.float() + s.float()).bfloat16()) @ w.t().contiguous())
    moe.device_error()


def test_a_step_captured(dev):
    # two graphs that share the library's scratch, replayed in turn with eager work between
    g = torch.Generator().manual_seed(3)
    halves, head = example.build(4, 256, 96, 16, 4, 100, g)
    ins = [[torch.randn(m, 256, generator=g).bfloat16().to(dev) for _ in "xr"] for m in (3, 16)]
    for x, r in ins:
        example.step(halves, head, x, r.clone())
    graphs, outs = [], []
    for x, r in ins:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(example.step(halves, head, x, r.clone()))
        graphs.append(graph)
    for seed in range(3):
        for (x, r), graph, out in zip(ins, graphs, outs):
            x.copy_(torch.randn(x.shape, generator=g).bfloat16())
            want = example.step(halves, head, x, r.clone())
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_caller_allocator(dev):
    # scratch from the caller's allocator: handed back after each call, the same bits
    from ubridge_amd import ops
    g = torch.Generator().manual_seed(1)
    halves, head = example.build(2, 256, 96, 16, 4, 100, g)
    x = torch.randn(12, 256, generator=g).bfloat16().to(dev)
    big = torch.randn(300, 2000, generator=g).bfloat16().to(dev)
    lin = mx.Linear(*mx.quantize(torch.randn(200, 2000, generator=g).to(dev)), 2000)
    w = torch.ones(2000, device=dev, requires_grad=True)

    def run():
        y = norm.RmsNorm(w)(big)
        return [example.step(halves, head, x, x.clone()), lin(big), torch.autograd.grad(y.float().sum(), [w])[0]]
    want = run()
    alloc = ops.TorchWorkspaceAllocator()
    ops.set_workspace_allocator(alloc)
    try:
        got = run()
        torch.cuda.synchronize()
    finally:
        ops.set_workspace_allocator(None)
    assert alloc.calls >= 3 and not alloc.live and ops.workspace_stats()[2] == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_main(dev, capsys, monkeypatch):
    monkeypatch.setattr("sys.argv", ["feed_forward.py", "--layers", "2", "--hidden", "256", "--inner", "96", "--experts", "8",
                                     "--topk", "2", "--vocab", "100"])
    example.main()
    assert "tokens" in capsys.readouterr().out


def test_graphs_of_one_stream_side_by_side(dev):
    # two graphs captured on one stream have scratch of their own each: replayed on two
    # streams at once, beside eager calls, all keep their bits
    from ubridge_amd import ops
    g = torch.Generator().manual_seed(5)
    halves, head = example.build(2, 256, 96, 16, 4, 100, g)
    layer = halves[1][1].layer
    lin = mx.Linear(*mx.quantize(torch.randn(200, 2000, generator=g).to(dev)), 2000)
    n = norm.RmsNorm(torch.rand(2000, generator=g).to(dev).requires_grad_())

    def run(x, lg, big, dy):
        w = n.weight
        return [layer.decode(x, lg), lin(big), torch.autograd.grad(n(big), [w], dy)[0]]
    E = layer.E
    ins = [[torch.randn(m, 256, generator=g).bfloat16().to(dev), torch.randn(m, E, generator=g).to(dev),
            torch.randn(300, 2000, generator=g).bfloat16().to(dev), torch.randn(300, 2000, generator=g).bfloat16().to(dev)]
           for m in (16, 16, 16)]
    want = [run(*i) for i in ins]
    want = [[t.clone() for t in w] for w in want]
    capture = torch.cuda.Stream()
    ops.release_workspace(capture)
    live = [ops.workspace_stats()[0]]
    graphs, outs = [], []
    for i in ins[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=capture):
            outs.append(run(*i))
        graphs.append(graph)
        live.append(ops.workspace_stats()[0])
    assert live[0] < live[1] < live[2], live
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(capture):
            got = run(*ins[2])
        torch.cuda.synchronize()
        for o, w in zip([*outs, got], want):
            assert all(torch.equal(a, b) for a, b in zip(o, w))
    del graphs, outs
    ops.release_workspace(capture)
    assert ops.workspace_stats()[0] == live[0]
