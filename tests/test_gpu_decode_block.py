"""The attention block's operators together, as examples/decode_block.py runs
them, against the same block in 64 bits over plain lists of keys and values.

Tolerance: between the two lie bf16 roundings (2^-9 of a value at most, half a
step) of q, k, v, the turned q and k, the attention's output and the result, and
where they move an activation across a border of its int8 code, one code of
254.  Norms add at most these: 7 * 2^-8 + 2^-7, below 2^-4.
"""
import importlib.util
import math
import os

import pytest
import torch

from conftest import ROOT
from ubridge_amd import kvcache, moe, rope

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location("decode_block", os.path.join(ROOT, "examples", "decode_block.py"))
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)


def linear64(lin, x):
    x = x.float()
    s = x.abs().amax(1, keepdim=True) / 127
    q = torch.round(x / s).double()
    return (q @ lin.w[:, :lin.K].double().t().contiguous()) * s.double() * lin.w_scale.double()


class Plain:
    """A layer's keys and values, one list a row."""

    def __init__(self, block, turn, rows):
        self.block, self.turn = block, turn
        self.k, self.v = [[] for _ in range(rows)], [[] for _ in range(rows)]

    def rotate(self, x, pos):
        a = pos * 2 * math.pi * self.turn.turns
        c, s = torch.cos(a), torch.sin(a)
        h = x.shape[-1] // 2
        p, q = x[..., :h], x[..., h:]
        return torch.cat([p * c - q * s, q * c + p * s], -1)

    def __call__(self, x, rows):
        b = self.block
        out = []
        y = linear64(b.qkv, x)
        for i, r in enumerate(rows):
            q, k, v = (z.view(-1, b.D) for z in y[i].split([b.Hq * b.D, b.Hkv * b.D, b.Hkv * b.D]))
            pos = len(self.k[r])
            self.k[r] = self.k[r] + [self.rotate(k, pos)]
            self.v[r] = self.v[r] + [v]
            K, V = torch.stack(self.k[r]), torch.stack(self.v[r])  # [n, Hkv, D]
            q = self.rotate(q, pos).view(b.Hkv, -1, b.D)
            o = [torch.softmax(q[h] @ K[:, h].t().contiguous() / b.D ** 0.5, -1) @ V[:, h] for h in range(b.Hkv)]
            out.append(torch.cat(o).flatten())
        return linear64(b.out, torch.stack(out))


def test_decode_with_samples(dev):
    g = torch.Generator().manual_seed(3)
    layers, hidden, Hq, Hkv, D, S = 2, 192, 4, 2, 32, 8
    blocks = [example.Block(hidden, Hq, Hkv, D, g) for _ in range(layers)]
    cache = kvcache.PagedCache(torch.full((layers, 2, 40, Hkv, S, D), float("nan"), device=dev).bfloat16(),
                               rows=8, width=5)
    turn = rope.Rope(D, base=10000.0)
    plain = [Plain(b, turn, 8) for b in blocks]
    ti = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)

    def both(rows, steps):
        for _ in range(steps):
            x = torch.randn(len(rows), hidden, generator=g).bfloat16().to(dev)
            # layer by layer on the same input, so that errors do not build up
            pos, slots = example.grow(cache, ti(rows))
            t, n = cache.tables[ti(rows).long()], cache.lens[ti(rows).long()]
            for layer, block in enumerate(blocks):
                got = block(x, cache, layer, turn, pos, slots, t, n).double()
                want = plain[layer](x, rows)
                assert float((got - want).norm() / want.norm()) < 2.0**-4
                x = torch.randn(len(rows), hidden, generator=g).bfloat16().to(dev)

    both([0, 1], 13)
    cache.fork(ti([0, 1, 0, 1]), ti([2, 3, 4, 5]))
    for p in plain:
        for s, d in ((0, 2), (1, 3), (0, 4), (1, 5)):
            p.k[d], p.v[d] = p.k[s], p.v[s]
    both([2, 3, 4, 5], 9)
    cache.free(ti([0, 3]))
    for p in plain:
        for d in (0, 3):
            p.k[d], p.v[d] = [], []
    used = int(cache.compact())
    assert used == int((cache.refs != 0).sum()) == int(cache.refs[:used].bool().sum())
    both([1, 2, 4, 5], 6)
    cache.fork(ti([2]), ti([0]))
    for p in plain:
        p.k[0], p.v[0] = p.k[2], p.v[2]
    both([0, 1, 2, 5], 5)
    moe.device_error()


def test_caller_allocator(dev):
    # scratch from the caller's allocator: handed back after each call, the same bits
    from ubridge_amd import attention, int8, ops
    g = torch.Generator().manual_seed(1)
    kv = torch.randn(1, 2, 300, 2, 8, 32, generator=g).bfloat16().to(dev)
    tables = torch.randperm(300, generator=g).int().view(2, 150).to(dev)
    lens = torch.tensor([1200, 777], dtype=torch.int32, device=dev)
    q = torch.randn(2, 8, 32, generator=g).bfloat16().to(dev)
    w = torch.randint(-127, 128, (96, 5000), generator=g, dtype=torch.int8)
    lin = int8.Linear(w.to(dev), torch.ones(96, device=dev))
    x = torch.randn(33, 5000, generator=g).to(dev)

    def run():
        c = kvcache.PagedCache(kv.clone(), rows=3, width=4)
        c.meta[:5] = 1
        c.lens[0], c.tables[0, :2] = 11, torch.tensor([0, 3], dtype=torch.int32)
        rows = torch.tensor([0, 1], dtype=torch.int32, device=dev)
        new = c.fork(rows[:1], rows[1:])
        n = c.compact()
        return [attention.paged_decode(q, kv[0, 0], kv[0, 1], tables, lens), lin(x), new, n, c.meta,
                c.kv.view(torch.int16)]

    want = run()
    alloc = ops.TorchWorkspaceAllocator()
    ops.set_workspace_allocator(alloc)
    try:
        got = run()
        torch.cuda.synchronize()
    finally:
        ops.set_workspace_allocator(None)
    assert alloc.calls >= 4 and not alloc.live and ops.workspace_stats()[2] == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))
