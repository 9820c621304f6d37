"""Rotary positions on the queries and keys of a decoder: half and interleaved
layouts, part of a head, contexts stretched linearly, by a larger base, by a
ramp over the frequencies ("yarn") or by bands of wavelengths.  The angles are
formed in 64 bits on the device, so positions may lie as far as a context
reaches without a table of sines; the rotation is f32."""
import math

import torch
from torch.autograd import forward_ad

from .native import _native, call


def frequencies(rot, base=10000.0, scaling=None):
    """(angle per position of the rot / 2 pairs, as floats of 64 bits; the
    factor on the rotated values).  scaling is None or one of

      kind="linear", factor                positions divided by factor
      kind="ntk", factor                   base times factor ** (rot / (rot - 2))
      kind="yarn", factor, original        pairs that turn fewer than `slow` times
                   [fast=32, slow=1]       over the original length divided by
                   [attention]             factor, those that turn more than `fast`
                                           times kept, a ramp between; values
                                           times attention, 0.1 ln(factor) + 1
      kind="bands", factor, original,      the same with a ramp in the number of
                    low, high              turns, from low to high
    """
    def need(*names):
        extra = set(scaling) - {"kind", *names}
        missing = [n for n in names if n not in scaling and n not in ("fast", "slow", "attention")]
        if extra or missing:
            raise ValueError(f"rope scaling {kind!r}: missing {missing}, unknown {sorted(extra)}")
        if not scaling["factor"] > 0:
            raise ValueError(f"rope scaling {kind!r}: factor {scaling['factor']}")

    i = range(rot // 2)
    factor = 1.0
    kind = scaling["kind"] if scaling else None
    if kind == "ntk":
        need("factor")
        base = base * scaling["factor"] ** (rot / (rot - 2.0)) if rot > 2 else base
    f = [base ** (-2.0 * k / rot) for k in i]
    if kind == "linear":
        need("factor")
        f = [x / scaling["factor"] for x in f]
    elif kind == "yarn":
        need("factor", "original", "fast", "slow", "attention")

        def turn(n):  # the pair that makes n turns over the original length
            return rot * math.log(scaling["original"] / (n * 2 * math.pi)) / (2 * math.log(base))
        low = max(math.floor(turn(scaling.get("fast", 32))), 0)
        high = min(math.ceil(turn(scaling.get("slow", 1))), rot - 1)
        ramp = [min(max((k - low) / max(high - low, 0.001), 0.0), 1.0) for k in i]
        f = [x / scaling["factor"] * r + x * (1 - r) for x, r in zip(f, ramp)]
        factor = scaling.get("attention")
        if factor is None:
            factor = 0.1 * math.log(scaling["factor"]) + 1.0
    elif kind == "bands":
        need("factor", "original", "low", "high")
        lo, hi = scaling["low"], scaling["high"]
        mix = [min(max((scaling["original"] * x / (2 * math.pi) - lo) / (hi - lo), 0.0), 1.0) for x in f]
        f = [x * (m + (1 - m) / scaling["factor"]) for x, m in zip(f, mix)]
    elif kind not in (None, "ntk"):
        raise ValueError(f"rope scaling kind {kind!r}")
    return f, factor


class Rope:
    """Rotary positions on the first `rot` elements of a head (even; the rest
    pass through).  Pairs are (x[i], x[i + rot / 2]), or neighbours when
    `interleaved`; see frequencies() for `base` and `scaling`.

    rope(q, k, positions) -> [q', k'] for q [T, Hq, D], k [T, Hkv, D] (f32, f16
    or bf16, any token and head strides) and positions int32 or int64 [T].  k
    may be None.  backward(dq, dk, positions) is the gradient by itself, the
    inverse turn.  Both are differentiable, any number of times and in forward
    mode: they are linear in q and k.
    """

    def __init__(self, rot, base=10000.0, interleaved=False, scaling=None, device="cuda"):
        if rot < 0 or rot % 2:
            raise ValueError(f"rope: rot={rot} must be even")
        self.rot, self.interleaved = rot, bool(interleaved)
        freqs, self.factor = frequencies(rot, base, scaling)
        self.turns = torch.tensor([f / (2 * math.pi) for f in freqs], dtype=torch.float64,
                                  device=device)

    def _run(self, q, k, positions, inverse, stream):
        return call(_native.rope, stream, q, k, positions, self.turns, self.rot, self.interleaved,
                    self.factor, inverse)

    def _turn(self, q, k, positions, inverse, stream):
        if _level() >= 0 or torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
            return list(_Turn.apply(q, k, positions, self, inverse, stream))
        return self._run(q, k, positions, inverse, stream)

    def forward(self, q, k, positions, stream=None):
        return self._turn(q, k, positions, False, stream)

    __call__ = forward

    def backward(self, dq, dk, positions, stream=None):
        """The gradients of q and k from those of the turned ones."""
        return self._turn(dq, dk, positions, True, stream)


def _level():
    return forward_ad._current_level  # (-1: not in forward mode)


def _stored(d):
    """A gradient or tangent that the kernel can read: expanded ones, and zeros
    that have no memory, written out."""
    if d is None or d.stride(-1) == 1 and not d._is_zerotensor():
        return d
    return torch.zeros(d.shape, dtype=d.dtype, device=d.device) if d._is_zerotensor() else d.contiguous()


class _Turn(torch.autograd.Function):
    """The turn, or the inverse one: each is the other's gradient, and its own
    derivative along q and k."""

    @staticmethod
    def forward(q, k, positions, rope, inverse, stream):
        return tuple(rope._run(q, k, positions, inverse, stream))

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, k, positions, ctx.rope, ctx.inverse, _ = inputs
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        ctx.keys = k is not None

    @staticmethod
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        dq, dk = ctx.rope._turn(_stored(dq), _stored(dk), positions, not ctx.inverse, None)
        return dq, dk, None, None, None, None

    @staticmethod
    def jvp(ctx, q, k, *_):
        (positions,) = ctx.saved_tensors
        k = _stored(k) if ctx.keys else None
        return tuple(ctx.rope._turn(_stored(q), k, positions, ctx.inverse, None))
