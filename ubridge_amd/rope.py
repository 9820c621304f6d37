"""Rotary positions on the queries and keys of a decoder: half and interleaved
layouts, part of a head, contexts stretched linearly, by a larger base, by a
ramp over the frequencies ("yarn") or by bands of wavelengths.  The angles are
formed in 64 bits on the device, so positions may lie as far as a context
reaches without a table of sines; the rotation is f32."""
import math

import torch

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
    may be None.  It is differentiable; backward(dq, dk, positions) is the
    gradient by itself, the inverse turn.
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

    def forward(self, q, k, positions, stream=None):
        if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
            return list(_Turn.apply(q, k, positions, self, stream))
        return self._run(q, k, positions, False, stream)

    __call__ = forward

    def backward(self, dq, dk, positions, stream=None):
        """The gradients of q and k from those of the turned ones."""
        return self._run(dq, dk, positions, True, stream)


class _Turn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, rope, stream):
        ctx.save_for_backward(positions)
        ctx.rope = rope
        return tuple(rope._run(q, k, positions, False, stream))

    @staticmethod
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        dq, dk = (None if d is None else d if d.stride(-1) == 1 else d.contiguous() for d in (dq, dk))
        dq, dk = ctx.rope._run(dq, dk, positions, True, None)
        return dq, dk, None, None, None
