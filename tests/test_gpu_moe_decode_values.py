"""The gated activations of FusedMoE.decode keep 16 bits and the range of f32 between its
two products.

Tolerance as in test_gpu_moe_decode.py, but that a is rounded to 2^-17 of itself (the
sum of two bf16: 2^-9 of what 2^-9 leaves, twice that allowed).
"""
import pytest
import torch

from test_gpu_moe_decode import make, routed

pytestmark = pytest.mark.gpu


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
            da = 1.1 * dg * (u.abs() + du) + s.abs() * du + a.abs() * (2.0**-17 + 2.0**-20)
            y[t] += p * (w2 * a).sum(1)
            tol[t] += p * ((w2.abs() * da).sum(1) * (1 + cI) + (cI + 2.0**-20) * (w2 * a).abs().sum(1))
    tol = tol * (1 + half) + half * y.abs() + tiny
    err = (got.double() - y).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    return y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T,E,k,H,I", [
    (1, 8, 2, 64, 96), (16, 128, 8, 256, 96), (16, 1, 1, 96, 32), (5, 1, 1, 64, 64), (16, 3, 2, 160, 224), (13, 4, 4, 96, 64),
    (16, 16, 16, 96, 224), (4, 2, 1, 512, 288), (9, 5, 3, 2080, 544), (16, 300, 16, 128, 32), (8, 32, 4, 4128, 96), (16, 48, 3, 4128, 224)])
def test_values(dev, T, E, k, H, I, q8, dtype):
    x, lg, layer = make(dev, T, E, k, H, I, dtype, q8)
    check(x, lg, layer, layer.decode(x, lg))


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T", [1, 16])
def test_activations_that_f16_does_not_hold(dev, T, q8):
    # gate and up of several hundreds: their product is past 65504, y is not
    x, lg, layer = make(dev, T, 12, 3, 256, 96, torch.float16, q8)
    x *= 400
    for t in (layer.s2,) if q8 else (layer.w2,):
        t *= 2.0**-10
    y = check(x, lg, layer, layer.decode(x, lg))
    assert float(y.abs().max()) < 6e4
    w13 = layer.w13[0].double() * (layer.s13[0].double()[:, None] if q8 else 1)
    g, u = (w13 @ x[0].double()).chunk(2)
    assert float((torch.nn.functional.silu(g) * u).abs().max()) > 65504
    # in bf16 too: a past 3e38 would be needed to lose any, and small ones keep their bits
    x, lg, layer = make(dev, T, 12, 3, 256, 96, torch.bfloat16, q8)
    x *= 2.0**-30
    for t in (layer.s2,) if q8 else (layer.w2,):
        t *= 2.0**60
    check(x, lg, layer, layer.decode(x, lg))


def test_infinite_results_stay_with_their_token(dev):
    # a of 1e13 and more: f32 holds it, f16 does not hold y; without a NaN anywhere
    x, lg, layer = make(dev, 6, 2, 2, 128, 64, torch.float16, False)
    clean = layer.decode(x, lg)
    x[3] *= 2.0**12
    got = layer.decode(x, lg)
    keep = [0, 1, 2, 4, 5]
    assert torch.equal(got[keep], clean[keep])
    y = check(x[keep], lg[keep], layer, got[keep])
    assert y.shape == (5, 128) and bool(torch.isinf(got[3]).any()) and not bool(torch.isnan(got[3]).any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("T,E,k,H,I", [(16, 6, 3, 2560, 96), (13, 3, 1, 4096, 160), (16, 16, 16, 2080, 32), (1, 8, 8, 4096, 224),
                                       (16, 2, 1, 7168, 32), (9, 64, 8, 2592, 96), (16, 4, 4, 5120, 64), (16, 1, 1, 4096, 32)])
def test_wide_results(dev, T, E, k, H, I, q8, dtype):
    # on both sides of where a workgroup takes 16 columns and 8 tokens of one expert
    x, lg, layer = make(dev, T, E, k, H, I, dtype, q8)
    check(x, lg, layer, layer.decode(x, lg))
