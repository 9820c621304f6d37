"""Derivatives of the rotation beyond the first: their structure on the CPU, with
the turn itself as its formula in 64 bits in the place of the kernel, and the
kernel's own on the device."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from ubridge_amd import rope


def formula(r, x, positions, inverse):
    x = x.double()
    a = positions.double().to(x.device)[:, None, None] * (2 * math.pi * r.turns.to(x.device))
    c, s = torch.cos(a) * r.factor, torch.sin(a) * r.factor * (-1 if inverse else 1)
    p, z = x[..., :r.rot // 2], x[..., r.rot // 2:r.rot]
    return torch.cat([p * c - z * s, z * c + p * s, x[..., r.rot:]], -1)


class Formula(rope.Rope):
    """Its kernel, as the kernel is to autograd: memory in, new memory out."""

    def _run(self, q, k, positions, inverse, stream):
        return [x if x is None else formula(self, x.detach(), positions, inverse) for x in (q, k)]


POS = torch.tensor([0, 3, 70000])


def inputs(*heads):
    g = torch.Generator().manual_seed(2)
    return [torch.randn(3, h, 10, dtype=torch.float64, generator=g).requires_grad_() for h in heads]


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("keys", [False, True])
def test_every_order(inverse, keys):
    r = Formula(8, device="cpu", scaling=dict(kind="yarn", factor=32.0, original=32768))

    def turn(q, k=None):
        y = (r.backward if inverse else r)(q, k, POS)
        return tuple(y) if keys else y[0]
    x = tuple(inputs(2, 1) if keys else inputs(2))
    assert torch.autograd.gradcheck(turn, x, check_forward_ad=True)
    assert torch.autograd.gradgradcheck(turn, x)


def test_one_input_only():
    r = Formula(8, device="cpu")
    q, k = (x.detach() for x in inputs(2, 1))
    with forward_ad.dual_level():
        for a, b in ((forward_ad.make_dual(q, k.expand(3, 2, 10)), k), (q, forward_ad.make_dual(k, 2 * k))):
            for x, y in zip((a, b), r(a, b, POS)):
                t, ty = forward_ad.unpack_dual(x).tangent, forward_ad.unpack_dual(y).tangent
                want = torch.zeros_like(y) if t is None else formula(r, t, POS, False)
                assert torch.equal(torch.zeros_like(y) if ty is None else ty, want)
        assert forward_ad.unpack_dual(r(q, None, POS)[0]).tangent is None
    # with a graph of k's alone, q's gradient is not asked for
    k.requires_grad_()
    y = r(q, k, POS)
    (g,) = torch.autograd.grad((y[1] ** 2).sum(), [k])
    assert torch.allclose(g, 2 * k, atol=1e-12)


def penalty(turn, q, k):
    """The gradients of the size of a gradient through the turn."""
    yq, yk = turn(q, k)
    grads = torch.autograd.grad((yq ** 3).sum() + (yk ** 3).sum(), [q, k], create_graph=True)
    return torch.autograd.grad(sum((x ** 2).sum() for x in grads), [q, k])


def test_penalty_on_the_cpu():
    r = Formula(8, device="cpu")
    q, k = inputs(2, 1)
    got = penalty(lambda q, k: r(q, k, POS), q, k)
    for a, b in zip(got, penalty(lambda q, k: [formula(r, x, POS, False) for x in (q, k)], q, k)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


@pytest.mark.gpu
def test_penalty(dev):
    # f32 against the formula in 64 bits.  Four turns and a dozen products lie between,
    # each good to some 2^-22 of values whose terms add up to at most some hundred:
    # norms within 2^-16
    r = rope.Rope(8)
    q, k = (x.detach().float().to(dev).requires_grad_() for x in inputs(2, 1))
    pos = POS.to(dev)
    got = penalty(lambda q, k: r(q, k, pos), q, k)
    q, k = (x.detach().double().requires_grad_() for x in (q, k))
    for a, b in zip(got, penalty(lambda q, k: [formula(r, x, pos, False) for x in (q, k)], q, k)):
        assert float((a.double() - b).norm()) <= 2.0**-16 * float(b.norm())


@pytest.mark.gpu
def test_forward_mode(dev):
    r = rope.Rope(8)
    q, k = (x.detach().float().to(dev) for x in inputs(2, 1))
    pos = POS.to(dev)
    near = lambda got, want: float((got.double() - want).norm()) <= 2.0**-20 * float(want.norm())
    with forward_ad.dual_level():
        for tangent in (torch.randn(3, 2, 10, device=dev), torch.randn(3, 10, 2, device=dev).transpose(1, 2),
                        torch.ones(1, device=dev).expand(3, 2, 10)):
            for turn, inverse in ((r, False), (r.backward, True)):
                y = turn(forward_ad.make_dual(q, tangent), k, pos)
                assert near(forward_ad.unpack_dual(y[0]).tangent, formula(r, tangent, pos, inverse))
                t = forward_ad.unpack_dual(y[1]).tangent
                assert t is None or not bool(t.any())
                assert torch.equal(forward_ad.unpack_dual(y[1]).primal, turn(q, k, pos)[1])
