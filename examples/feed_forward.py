"""The norms and feed-forward halves of a quantized decoder's layers, decoding and
training.

Per layer: the attention half's output joins the residual stream and is normed (one
launch), then either a dense feed-forward (the norm rounds its result to blocks for
the 4-bit gate and up projection, SiLU, the 4-bit down projection) or a mixture of
experts for a few tokens (two launches).  A norm in training gives its gradients.

    python examples/feed_forward.py [--layers 4] [--tokens 8]
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from ubridge_amd import int8, moe, mx, norm  # noqa: E402


class Dense:
    """Gate, up and down projections in 4-bit blocks; activations in blocks of `act`."""

    def __init__(self, w13, w2, act="fp8"):
        self.w13 = mx.Linear(*mx.quantize(w13), w13.shape[1], activations=act)
        self.w2 = mx.Linear(*mx.quantize(w2), w2.shape[1], activations=act)
        self.act = act

    def __call__(self, n, x, residual):
        """(this half's output, the residual stream): x joins it ahead of the norm n."""
        codes, scales, h = n(x, residual, quant=self.act, residual_out=residual)
        gate_up = self.w13.codes(codes, scales, x.dtype)
        return self.w2(moe.silu_and_mul(gate_up)), h


class Experts:
    """A router and int8 experts for up to 16 tokens."""

    def __init__(self, router, w13, w2, s13, s2, topk):
        self.router = router
        self.layer = moe.FusedMoE(w13, w2, s13, s2, topk=topk)

    def __call__(self, n, x, residual):
        y, h = n(x, residual, residual_out=residual)
        return self.layer.decode(y, y.float() @ self.router), h


class Head:
    """The last norm, in int8 codes for an int8 projection."""

    def __init__(self, w, w_scale):
        self.linear = int8.Linear(w, w_scale)

    def __call__(self, n, x, residual):
        codes, scales, _ = n(x, residual, quant="int8")
        return self.linear.codes(codes, scales, x.dtype)


def build(layers, hidden, inner, experts, topk, vocab, generator, device="cuda"):
    """[(norm, half)] with dense and expert halves in turn, and the head."""
    def rand(*shape):
        return torch.randn(*shape, generator=generator).to(device) * shape[-1] ** -0.5

    def gain():
        return norm.RmsNorm((1 + 0.1 * torch.randn(hidden, generator=generator)).bfloat16().to(device))

    def codes(*shape):
        return torch.randint(-127, 128, shape, generator=generator, dtype=torch.int8).to(device)

    def scale(rows, k):
        return torch.full(rows, 1 / (73 * k ** 0.5), device=device)
    halves = []
    for i in range(layers):
        if i % 2 == 0:
            half = Dense(rand(2 * inner, hidden).bfloat16(), rand(hidden, inner).bfloat16())
        else:
            half = Experts(rand(hidden, experts), codes(experts, 2 * inner, hidden), codes(experts, hidden, inner),
                           scale((experts, 2 * inner), hidden).bfloat16(), scale((experts, hidden), inner).bfloat16(), topk)
        halves.append((gain(), half))
    return halves, (gain(), Head(codes(vocab, hidden), scale((vocab,), hidden)))


def step(halves, head, x, residual):
    """Logits of one pass; the residual stream is written in place."""
    for n, half in halves:
        x, residual = half(n, x, residual)
    n, last = head
    return last(n, x, residual)


def main():
    p = argparse.ArgumentParser()
    for name, default in (("layers", 4), ("hidden", 2048), ("inner", 768), ("experts", 128), ("topk", 8),
                          ("vocab", 9001), ("tokens", 8)):
        p.add_argument("--" + name, type=int, default=default)
    a = p.parse_args()
    g = torch.Generator().manual_seed(0)
    halves, head = build(a.layers, a.hidden, a.inner, a.experts, a.topk, a.vocab, g)
    x = torch.randn(a.tokens, a.hidden, generator=g).bfloat16().cuda()
    r = torch.randn(a.tokens, a.hidden, generator=g).bfloat16().cuda()
    for _ in range(5):
        y = step(halves, head, x, r.clone())
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(50):
        y = step(halves, head, x, r.clone())
    torch.cuda.synchronize()
    t = (time.perf_counter() - t) / 50
    # a training step of one norm
    w = torch.ones(a.hidden, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    xt, rt = (torch.randn(2048, a.hidden, generator=g).bfloat16().cuda().requires_grad_() for _ in "xr")
    n, h = norm.RmsNorm(w)(xt, rt)
    (n.float().square().mean() + h.float().mean()).backward()
    assert all(bool(torch.isfinite(v).all()) for v in (y, w.grad, xt.grad, rt.grad))
    print(f"{a.tokens} tokens, {a.layers} feed-forward halves and the head: {t * 1e6:.0f} us")


if __name__ == "__main__":
    main()
