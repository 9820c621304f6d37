"""The mixture-of-experts layer for a few tokens against its definition in 64 bits.

Tolerance, per output: f32 sums of K products lose at most (K / 32 + 24) * 2^-23 of
their sum of magnitudes (instructions of 32 products, 16 wavefronts' sums, scales);
of g and u that passes to a by |silu'| <= 1.1, |u|, |silu(g)|; exp and the quotient
cost 2^-20 of a, which is rounded to T (half a step, and a smallest denormal); routed
weights have 2^-20.  All of it passes through the second product, whose own sum and
rounding follow.
"""
import math

import pytest
import torch

from ubridge_amd import moe

pytestmark = pytest.mark.gpu


def make(dev, T, E, k, H, I, dtype, q8, norm=True, seed=0, logits=torch.float32):
    g = torch.Generator().manual_seed(seed + T + E + H + I)
    x = torch.randn(T, H, generator=g).to(dtype)
    lg = torch.randn(T, E, generator=g).to(logits)
    if q8:
        w13 = torch.randint(-128, 128, (E, 2 * I, H), generator=g, dtype=torch.int8)
        w2 = torch.randint(-128, 128, (E, H, I), generator=g, dtype=torch.int8)
        s13 = ((torch.rand(E, 2 * I, generator=g) + 0.5) / (73 * H**0.5)).to(dtype)
        s2 = ((torch.rand(E, H, generator=g) + 0.5) / (73 * I**0.5)).to(dtype)
    else:
        w13 = (torch.randn(E, 2 * I, H, generator=g) * H**-0.5).to(dtype)
        w2 = (torch.randn(E, H, I, generator=g) * I**-0.5).to(dtype)
        s13 = s2 = None
    d = [None if t is None else t.to(dev) for t in (x, lg, w13, w2, s13, s2)]
    return d[0], d[1], moe.FusedMoE(*d[2:], topk=k, renormalize=norm)


def routed(lg, k, norm):
    """per token {expert: weight}"""
    out = []
    for row in lg.double().cpu():
        ok = [e for e in range(len(row)) if row[e] > -math.inf]  # (a NaN is not)
        order = sorted(ok, key=lambda e: (-float(row[e]), e))[:k]
        if not order:
            out.append({})
            continue
        p = torch.exp(row - row[order[0]])
        total = sum(float(p[e]) for e in (order if norm else ok))
        out.append({e: float(p[e]) / total for e in order})
    return out


def check(x, lg, layer, got):
    T, H = x.shape
    dtype = x.dtype
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    I = layer.w2.shape[2]
    cH, cI = (H / 32 + 24) * 2.0**-23, (I / 32 + 24) * 2.0**-23
    y = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    tol = torch.zeros_like(y)
    for t, chosen in enumerate(routed(lg, layer.topk, layer.renormalize)):
        for e, p in chosen.items():
            w13, w2 = layer.w13[e].double(), layer.w2[e].double()
            if layer.s13 is not None:
                w13, w2 = w13 * layer.s13[e].double()[:, None], w2 * layer.s2[e].double()[:, None]
            xd = x[t].double()
            gu, mag = (w13 * xd).sum(1), (w13 * xd).abs().sum(1) * cH
            g, u, dg, du = gu[:I], gu[I:], mag[:I], mag[I:]
            s = g * torch.sigmoid(g)
            a = s * u
            da = 1.1 * dg * (u.abs() + du) + s.abs() * du + a.abs() * (half + 2.0**-20) + tiny
            y[t] += p * (w2 * a).sum(1)
            tol[t] += p * ((w2.abs() * da).sum(1) * (1 + cI) + (cI + 2.0**-20) * (w2 * a).abs().sum(1))
    tol = tol * (1 + half) + half * y.abs() + tiny
    err = (got.double() - y).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    return y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T,E,k,H,I,norm", [
    (1, 1, 1, 32, 32, True), (1, 8, 2, 64, 96, True), (3, 5, 5, 96, 32, False), (2, 64, 6, 160, 64, True),
    (16, 128, 8, 256, 96, True), (9, 130, 4, 288, 160, False), (16, 4, 1, 512, 64, True), (7, 300, 16, 128, 32, True),
    (8, 1024, 3, 64, 32, True), (5, 16, 3, 1056, 544, True), (16, 16, 16, 96, 224, False)])
def test_decode(dev, T, E, k, H, I, norm, q8, dtype):
    x, lg, layer = make(dev, T, E, k, H, I, dtype, q8, norm)
    check(x, lg, layer, layer.decode(x, lg))


@pytest.mark.parametrize("T,E,k,H,I,q8", [(1, 16, 4, 4096, 768, True), (4, 8, 2, 4096, 1024, False), (2, 8, 2, 7168, 2048, True),
                                          (3, 8, 2, 8224, 96, False), (1, 4, 2, 8192, 64, True), (16, 128, 8, 2048, 768, True)])
def test_decode_large(dev, T, E, k, H, I, q8):
    x, lg, layer = make(dev, T, E, k, H, I, torch.bfloat16, q8)
    check(x, lg, layer, layer.decode(x, lg))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,H,I,q8", [(16, 48, 3, 4128, 224, False), (16, 40, 4, 4160, 256, True), (9, 64, 8, 5152, 192, False),
                                          (2, 32, 16, 6176, 288, True), (7, 48, 8, 4128, 224, False), (11, 6, 3, 3552, 160, False),
                                          (16, 6, 3, 2080, 160, False), (13, 6, 3, 4064, 160, True)])
def test_decode_rows_in_pieces(dev, T, E, k, H, I, q8, dtype):
    x, lg, layer = make(dev, T, E, k, H, I, dtype, q8)
    check(x, lg, layer, layer.decode(x, lg))


@pytest.mark.parametrize("logits", [torch.float32, torch.float16, torch.bfloat16])
def test_against_forward(dev, logits):
    # the same layer by its three launches, whose gate, up, weights and rows are rounded
    # to T: four more half steps along the way, each at most of the sum of magnitudes,
    # which is about sqrt(k I) times the result: compared in norm, by four times a step
    x, lg, layer = make(dev, 12, 32, 4, 512, 256, torch.bfloat16, True, logits=logits)
    a, b = layer.decode(x, lg).double(), layer(x, lg).double()
    assert float((a - b).norm() / b.norm()) < 4 * 2.0**-7
    check(x, lg, layer, layer.decode(x, lg))


def test_ties_and_masks(dev):
    x, lg, layer = make(dev, 8, 40, 4, 64, 32, torch.float16, True)
    lg[0] = 0.0                     # all equal: the lowest four
    lg[1] = -math.inf               # nothing left
    lg[2] = -math.inf
    lg[2, 7], lg[2, 30] = 1.0, 2.0  # fewer than k
    lg[3] = math.nan                # nothing either
    lg[4, ::2] = math.nan
    lg[5] = torch.finfo(torch.float32).min  # masked by the lowest value: ordinary numbers
    lg[5, 33] = 3.0
    lg[6] = 200.0 * torch.arange(40, device=dev)  # weights that underflow
    y = layer.decode(x, lg)
    check(x, lg, layer, y)
    assert bool((y[1] == 0).all()) and bool((y[3] == 0).all())
    y = layer.decode(x[1:2], lg[1:2])  # no expert at all
    assert bool((y == 0).all())
    layer.renormalize = False
    check(x, lg, layer, layer.decode(x, lg))


def test_rows_apart(dev):
    # a token's NaN and infinities stay its own, also where it shares its experts
    x, lg, layer = make(dev, 6, 4, 2, 128, 64, torch.bfloat16, False)
    y = layer.decode(x, lg)
    x2 = x.clone()
    x2[2, 5], x2[4, 100] = math.nan, math.inf
    z = layer.decode(x2, lg)
    keep = [0, 1, 3, 5]
    assert torch.equal(z[keep], y[keep]) and bool(torch.isnan(z[2]).all())
    # one by one: the same products in another order of experts and steps
    for t in keep:
        check(x[t:t + 1], lg[t:t + 1], layer, layer.decode(x[t:t + 1], lg[t:t + 1]))


def test_views_streams_bits_and_refusals(dev):
    x, lg, layer = make(dev, 5, 16, 3, 96, 64, torch.bfloat16, True)
    y = layer.decode(x, lg)
    for _ in range(3):
        assert torch.equal(layer.decode(x, lg), y)
    assert torch.equal(layer.decode(torch.cat([x, x], 1)[:, :96], torch.cat([lg, lg], 1)[:, :16]), y)
    odd = torch.empty(5 * 96 + 1, device=dev, dtype=x.dtype)[1:].view(5, 96).copy_(x)
    assert torch.equal(layer.decode(odd, lg), y)
    assert layer.decode(x[:0], lg[:0]).shape == (0, 96)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = layer.decode(x, lg, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, y)
    big, blg, _ = make(dev, 17, 16, 3, 96, 64, torch.bfloat16, True)
    f = moe.FusedMoE
    for call in (lambda: layer.decode(big, blg), lambda: layer.decode(x.float(), lg), lambda: layer.decode(x.half(), lg),
                 lambda: layer.decode(x, lg[:, :8]), lambda: layer.decode(x[:, :64], lg), lambda: layer.decode(x, lg[:2]),
                 lambda: layer.decode(x.cpu(), lg), lambda: layer.decode(x, lg.double()),
                 lambda: f(layer.w13, layer.w2, topk=3).decode(x, lg),
                 lambda: f(layer.w13, layer.w2, layer.s13.float(), layer.s2.float(), topk=3).decode(x, lg),
                 lambda: f(layer.w13, layer.w2, layer.s13, layer.s2, topk=17).decode(x, lg),
                 lambda: f(layer.w13[:, :40], layer.w2, layer.s13, layer.s2, topk=3).decode(x, lg)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("T", [1, 13])
def test_graph(dev, T):
    x, lg, layer = make(dev, T, 32, 4, 256, 96, torch.float16, True)
    layer.decode(x, lg)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.decode(x, lg)
    for seed in range(1, 4):
        a, b, _ = make(dev, T, 32, 4, 256, 96, torch.float16, True, seed=seed)
        x.copy_(a), lg.copy_(b)
        want = layer.decode(x, lg)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("q8", [True, False])
def test_weights_past_32_bits(dev, q8):
    # the last experts of 4.3e9 weights give what a layer of these alone gives
    E, H, I = (64, 16384, 2048) if q8 else (40, 16384, 2048)
    g = torch.Generator(device=dev).manual_seed(1)
    kw = dict(device=dev, generator=g)
    if q8:
        w13, w2 = (torch.randint(-127, 128, s, dtype=torch.int8, **kw) for s in ((E, 2 * I, H), (E, H, I)))
        s13, s2 = (torch.rand(*s, **kw).half() * 1e-3 for s in ((E, 2 * I), (E, H)))
    else:
        w13, w2 = (torch.empty(*s, device=dev, dtype=torch.float16).normal_(generator=g).mul_(s[-1] ** -0.5)
                   for s in ((E, 2 * I, H), (E, H, I)))
        s13 = s2 = None
    x = torch.randn(3, H, **kw).half()
    lg = torch.full((3, E), -math.inf, device=dev)
    lg[:, -4:] = torch.randn(3, 4, **kw)
    y = moe.FusedMoE(w13, w2, s13, s2, topk=2).decode(x, lg)
    part = [t if t is None else t[-4:].contiguous() for t in (w13, w2, s13, s2)]
    assert torch.equal(y, moe.FusedMoE(*part, topk=2).decode(x, lg[:, -4:]))
