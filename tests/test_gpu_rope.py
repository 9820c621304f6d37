"""Rotary positions and the fused store into cache pages against the formula in
64 bits.

Tolerances.  The sine and cosine are within 2^-23 of their values (the angle's
remainder and each Taylor sum round a few times at 2^-24 and below 1), each
product and the sum round at 2^-24, so a turned value is off by at most
2^-21 (|a| + |b|) factor before it is rounded once to the output type.
"""
import math

import numpy as np
import pytest
import torch

from ubridge_amd import kvcache, moe, rope

pytestmark = pytest.mark.gpu

SCALINGS = [None, dict(kind="linear", factor=4.0), dict(kind="ntk", factor=4.0),
            dict(kind="yarn", factor=32.0, original=32768),
            dict(kind="bands", factor=8.0, low=1.0, high=4.0, original=8192)]


def turn64(x, pos, r, inverse=False):
    """The formula in 64 bits on [T, H, D], and the size its errors scale with."""
    rot, inter = r.rot, r.interleaved
    a = pos.double().cpu()[:, None, None] * (2 * math.pi * r.turns.cpu())
    c, s = torch.cos(a) * r.factor, torch.sin(a) * r.factor * (-1 if inverse else 1)
    y = x.double().cpu().clone()
    size = torch.zeros_like(y)
    lo = slice(0, rot, 2) if inter else slice(0, rot // 2)
    hi = slice(1, rot, 2) if inter else slice(rot // 2, rot)
    p, q = y[..., lo].clone(), y[..., hi].clone()
    y[..., lo], y[..., hi] = p * c - q * s, q * c + p * s
    size[..., lo] = size[..., hi] = (p.abs() + q.abs()) * r.factor
    return y, size


def near(got, want, size, dtype):
    half = 0.0 if dtype is None else torch.finfo(dtype).eps / 2
    tol = half * want.abs() + (1 + half) * 2.0**-21 * size
    if dtype is not None:
        tol = tol + torch.finfo(dtype).smallest_normal * half
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def heads(g, T, Hq, Hkv, D, dtype, dev, pad=0):
    """q, k, v as views of one projection (rows padded by `pad` elements)."""
    x = torch.randn(T, (Hq + 2 * Hkv) * D + pad, generator=g).to(dtype).to(dev)
    return [y.unflatten(1, (-1, D)) for y in x[:, :(Hq + 2 * Hkv) * D].split([Hq * D, Hkv * D, Hkv * D], 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot,pad", [
    (1, 1, 1, 2, 2, 0), (1, 8, 2, 64, 64, 0), (7, 3, 1, 40, 26, 3), (33, 4, 4, 80, 80, 1),
    (5, 6, 2, 96, 0, 0), (300, 2, 1, 128, 96, 0), (3, 16, 16, 256, 254, 5), (9, 1, 1, 7, 4, 0),
    (2, 40, 8, 192, 192, 8), (1100, 1, 1, 64, 2, 0), (2, 3, 1, 1000, 600, 0), (3, 2, 2, 1001, 1000, 1),
    (1, 1, 1, 4096, 4096, 0), (4, 5, 3, 130, 18, 0), (6, 2, 1, 70, 66, 2)])
def test_turn(dev, dtype, inter, T, Hq, Hkv, D, rot, pad):
    g = torch.Generator().manual_seed(T + D + rot)
    q, k, _ = heads(g, T, Hq, Hkv, D, dtype, dev, pad)
    pos = torch.randint(0, 5000, (T,), generator=g)
    r = rope.Rope(rot, base=500000.0, interleaved=inter)
    for p in (pos.to(dev), pos.int().to(dev)):
        for got, x in zip(r(q, k, p), (q, k)):
            near(got, *turn64(x, pos, r), dtype)
    for got, x in zip(r.backward(q, k, pos.to(dev)), (q, k)):
        near(got, *turn64(x, pos, r, inverse=True), dtype)


@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: s["kind"] if s else "none")
def test_far_positions(dev, scaling):
    # f32 inputs and positions up to 2^40: every bit of the angle counts
    g = torch.Generator().manual_seed(3)
    q, k, _ = heads(g, 64, 2, 1, 128, torch.float32, dev)
    pos = torch.cat([torch.arange(8), 2 ** torch.arange(8, 20), 2**20 + torch.arange(-4, 4),
                     torch.randint(0, 1 << 20, (36,), generator=g)])
    r = rope.Rope(128, base=500000.0, scaling=scaling)
    for got, x in zip(r(q, k, pos.to(dev)), (q, k)):
        near(got, *turn64(x, pos, r), torch.float32)


def test_negative_position_turns_back(dev):
    g = torch.Generator().manual_seed(4)
    q, k, _ = heads(g, 16, 2, 2, 64, torch.float32, dev)
    pos = torch.arange(-16, 0)
    r = rope.Rope(64)
    near(r(q, None, pos.to(dev))[0], *turn64(q, pos, r), torch.float32)
    assert r(q, None, pos.to(dev))[1] is None


def test_gradient(dev):
    # against the inverse turn's formula, and against differences of the turn
    g = torch.Generator().manual_seed(5)
    q, k, _ = (x.clone().requires_grad_() for x in heads(g, 6, 3, 1, 32, torch.float32, dev))
    pos = torch.randint(0, 9000, (6,), generator=g)
    r = rope.Rope(24, scaling=SCALINGS[3])
    dq, dk = torch.randn(6, 3, 32, generator=g).to(dev), torch.randn(6, 1, 32, generator=g).to(dev)
    yq, yk = r(q, k, pos.to(dev))
    gq, gk = torch.autograd.grad([yq, yk], [q, k], [dq, dk])
    for got, d in ((gq, dq), (gk, dk)):
        near(got, *turn64(d, pos, r, inverse=True), torch.float32)
    # the turn is linear: <turn(x + h e) - turn(x), d> / h = gradient . e, h = 1
    e = torch.randn(6, 3, 32, generator=g).to(dev)
    with torch.no_grad():
        diff = ((r(q + e, k, pos.to(dev))[0].double() - yq.double()) * dq.double()).sum()
    want = (gq.double() * e.double()).sum()
    # 576 terms, each off by at most 2^-21 of values below ~40
    assert abs(float(diff - want)) < 576 * 40 * 2.0**-21
    # the gradient of an expanded output, and of one input only
    (g1,) = torch.autograd.grad(r(q, k, pos.to(dev))[0].sum(), [q])
    near(g1, *turn64(torch.ones(6, 3, 32), pos, r, inverse=True), torch.float32)


def test_refusals(dev):
    q = torch.zeros(4, 2, 64, device=dev)
    pos = torch.arange(4, device=dev)
    r = rope.Rope(64)
    with pytest.raises(ValueError):
        rope.Rope(63)
    for args in ((q.cpu(), None, pos), (q, q.half(), pos), (q, None, pos[:3]), (q, None, pos.float()),
                 (q[..., :32], None, pos), (q[0], None, pos), (q, q[:3], pos),
                 (q, q.transpose(1, 2), pos), (q.double(), None, pos),
                 (q, None, torch.arange(8, device=dev)[::2])):
        with pytest.raises(ValueError):
            r(*args)
    qo, ko = r(q[:0], q[:0], pos[:0])
    assert qo.shape == (0, 2, 64) and ko.shape == (0, 2, 64)


def _e4m3_bounds(x, tol):
    """e4m3 values of x - tol and x + tol (saturating)."""
    out = []
    for y in (x - tol, x + tol):
        out.append(y.clamp(-448, 448).to(torch.float8_e4m3fn).double())
    return out


@pytest.mark.parametrize("dtype,cache", [("f16", "f16"), ("bf16", "bf16"), ("bf16", "e4m3"),
                                         ("f32", "e4m3"), ("f16", "e4m3")])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot,S", [(1, 8, 2, 128, 128, 16), (37, 3, 3, 80, 50, 24),
                                              (130, 2, 1, 40, 40, 1), (5, 7, 1, 256, 64, 64),
                                              (600, 1, 1, 64, 64, 8)])
def test_append(dev, dtype, cache, inter, T, Hq, Hkv, D, rot, S):
    DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
          "e4m3": torch.float8_e4m3fn}
    g = torch.Generator().manual_seed(T + D)
    q, k, v = heads(g, T, Hq, Hkv, D, DT[dtype], dev)
    pos = torch.randint(0, 1 << 20, (T,), generator=g)
    L, P = 2, (T + S - 1) // S + 3
    kv = torch.randn(L, 2, P, Hkv, S, D, generator=g).to(DT[cache]).to(dev)
    before = kv.view(torch.uint8 if cache == "e4m3" else kv.dtype).clone()
    slots = torch.randperm(P * S, generator=g)[:T]
    slots[T // 2] = -1  # (a padding token: stored nowhere)
    ks = vs = None
    if cache == "e4m3":
        ks, vs = (torch.rand(Hkv, generator=g).to(dev) * 0.05 + 0.001 for _ in "kv")
    c = kvcache.PagedCache(kv, rows=1, width=1, k_scale=ks, v_scale=vs)
    r = rope.Rope(rot, base=500000.0, interleaved=inter, scaling=SCALINGS[4])
    near(c.append(1, q, k, v, slots.to(dev), positions=pos.to(dev), rope=r), *turn64(q, pos, r), DT[dtype])
    live = slots >= 0
    page, at = slots[live] // S, slots[live] % S
    kt, size = turn64(k, pos, r)
    got_k, got_v = (kv[1, i].float().cpu()[page, :, at].double() for i in (0, 1))
    kt, size, vt = kt[live], size[live], v.double().cpu()[live]
    if cache == "e4m3":
        # the stored code lies between those of the value's error bounds
        kt, size = kt / ks.double().cpu()[:, None], size / ks.double().cpu()[:, None]
        lo, hi = _e4m3_bounds(kt, 2.0**-21 * size + 2.0**-23 * kt.abs())
        assert bool(((got_k >= lo) & (got_k <= hi)).all())
        want = (v.float().cpu()[live] / vs.cpu()[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        assert torch.equal(got_v, want.double())
    else:
        near(got_k, kt, size, DT[cache])
        assert torch.equal(got_v, vt)
    # nothing else changed
    after = kv.view(before.dtype).clone()
    a, b = (x[1].transpose(2, 3).reshape(2, P * S, Hkv, D) for x in (after, before))
    rest = torch.ones(P * S, dtype=torch.bool)
    rest[slots[live]] = False
    rest = rest.to(dev)
    assert torch.equal(a[:, rest], b[:, rest]) and torch.equal(after[0], before[0])


def test_append_without_rope_and_special_values(dev):
    g = torch.Generator().manual_seed(8)
    kv = torch.zeros(1, 2, 4, 1, 8, 8, device=dev).to(torch.float8_e4m3fn)
    c = kvcache.PagedCache(kv, rows=1, width=4)
    k = torch.randn(3, 1, 8, generator=g).to(dev).half()
    v = torch.tensor([float("nan"), float("inf"), -float("inf"), 1e4, -1e4, 0.0, 2.0**-9, 2.0**-11],
                     device=dev).half().expand(3, 1, 8).contiguous()
    q = torch.zeros(3, 2, 8, device=dev)
    assert c.append(0, q, k, v, torch.tensor([0, 9, 31], device=dev)) is q
    got = kv[0, 1].float()[[0, 1, 3], 0, [0, 1, 7]]
    assert bool(got[:, 0].isnan().all())
    assert torch.equal(got[:, 1:], torch.tensor([448.0, -448, 448, -448, 0, 2.0**-9, 0], device=dev).expand(3, 7))
    assert torch.equal(kv[0, 0].float()[[0, 1, 3], 0, [0, 1, 7]], k[:, 0].float().to(torch.float8_e4m3fn).float())
    moe.device_error()
    # a slot past the cache: reported, the others stored
    c.append(0, None, k, v, torch.tensor([32, 2, -5], device=dev))
    with pytest.raises(Exception, match="out of range"):
        moe.device_error()
    moe.device_error()
    assert torch.equal(kv[0, 0, 0, 0, 2].float(), k[1, 0].float().to(torch.float8_e4m3fn).float())


def test_append_refusals(dev):
    kv = torch.zeros(2, 2, 4, 2, 8, 16, device=dev, dtype=torch.bfloat16)
    c = kvcache.PagedCache(kv, rows=1, width=4)
    k = torch.zeros(3, 2, 16, device=dev, dtype=torch.bfloat16)
    s = torch.arange(3, device=dev)
    r = rope.Rope(16)
    for bad in (dict(layer=2), dict(layer=-1), dict(k=k.half()), dict(v=k[:2]), dict(slots=s.int()),
                dict(slots=s[:2]), dict(rope=r), dict(positions=s), dict(k=k.cpu()),
                dict(rope=rope.Rope(18), positions=s), dict(rope=r, positions=s, q=k.float()),
                dict(k=k[:, :1], v=k[:, :1]), dict(k=k.half(), v=k.half())):
        args = dict(dict(layer=0, q=k, k=k, v=k, slots=s, positions=None, rope=None), **bad)
        with pytest.raises(ValueError):
            c.append(**args)
    assert c.append(0, k[:0], k[:0], k[:0], s[:0], positions=s[:0], rope=r).shape == (0, 2, 16)
    assert not bool(kv.any())


def test_append_has_no_gradient(dev):
    kv = torch.zeros(1, 2, 4, 1, 8, 16, device=dev, dtype=torch.bfloat16)
    c = kvcache.PagedCache(kv, rows=1, width=4)
    q, k, v = (torch.ones(2, 1, 16, device=dev, dtype=torch.bfloat16, requires_grad=True) for _ in "qkv")
    slots = torch.arange(2, device=dev)
    assert not c.append(0, q, k, v, slots, slots, rope.Rope(16)).requires_grad
    assert not c.kv.requires_grad
    assert c.append(0, q, k, v, slots) is q  # without a rotation q is not touched
