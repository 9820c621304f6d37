"""Microscaled blocks: 32 consecutive values under one power of two, elements of 4
bits (e2m1, "fp4") or 8 (e4m3, "fp8"); a linear whose weight is held in 4-bit blocks.
None of it has a gradient: inputs that ask for one, or have a tangent, are refused.

Rows of C elements are stored as ld = C rounded up to 128 of them, zero past C:
codes uint8 [..., ld / 2] (two a byte, the even one low; "fp8": [..., ld]) and
scales uint8 [..., ld / 32], 127 + the block's exponent (255: its values are NaN)."""
import torch

from .native import _native, call
from .ops import _DT_CODE, _need_cuda

_BITS = {"fp4": 4, "fp8": 8}


def _bits(fmt):
    if fmt not in _BITS:
        raise ValueError(f"mx: format {fmt!r} (one of {list(_BITS)})")
    return _BITS[fmt]


def quantize(x, fmt="fp4", stream=None):
    """x [..., C] f32, f16 or bf16 -> (codes, scales).  A block's exponent is
    floor(log2 amax) - 2 ("fp8": - 8), at least -127; values go to the nearest
    element, ties to even, those past the largest (6, 448 times the power) to it.  A
    block that holds an infinity or a NaN becomes NaN."""
    return call(_native.mx_quantize, stream, x, _bits(fmt))


def dequantize(codes, scales, C, dtype=torch.bfloat16, stream=None):
    """The values [..., C] that codes and scales of quantize() stand for, rounded to
    dtype.  The format follows from the sizes."""
    if dtype not in _DT_CODE:
        raise ValueError(f"mx.dequantize: dtype {dtype}")
    fmt = 4 if codes.shape[-1:] == (-(-C // 128) * 64,) else 8
    return call(_native.mx_dequantize, stream, codes, scales, C, _DT_CODE[dtype], fmt)


class Linear:
    """y = a @ w.T + bias over 4-bit blocks w (codes and scales of quantize(weight [N,
    K], "fp4"), or a checkpoint's) with x rounded to blocks by the call: a are the values
    of quantize(x, activations), "fp4" or "fp8".

    x is f32, f16 or bf16 [..., K] and y [..., N] has its type; sums are f32, bias f32
    [N] or None.  exact=False, of 8-bit activations, f16 or bf16 results and more than 16
    tokens: one matrix product in place of two, which drops addends 2 ** -13 below the
    largest of their neighbours (at most 2 ** -10 of the sum of magnitudes).  `out`, if given, overlaps no input and asks for no gradient.  A block of NaN, in a row of x or
    of w, makes that row's results NaN.  The weight is laid out once: the tensors given
    are not kept.  codes(a, scales, dtype) takes activations that are in blocks already
    (norm.RmsNorm's), and gives y of dtype.
    """

    def __init__(self, codes, scales, K, bias=None, activations="fp4", exact=True):
        _need_cuda(codes, scales, bias)
        self.bits, self.exact = _bits(activations), exact
        if codes.dim() != 2:
            raise ValueError("mx.Linear takes a weight [N, K] in blocks")
        self.N, self.K = codes.shape[0], K
        if bias is not None and (bias.shape != (self.N,) or bias.dtype != torch.float32):
            raise ValueError(f"mx.Linear: bias must be float32 [{self.N}]")
        self.bias = None if bias is None else bias.contiguous()
        self.w, self.w_scales = call(_native.mx_pack, None, codes.contiguous(), scales.contiguous(), K)

    def forward(self, x, out=None, stream=None):
        return call(_native.mx_linear, stream, x, None, self.w, self.w_scales, self.bias, self.K, self.N, self.bits,
                    0, out, not self.exact)

    __call__ = forward

    def codes(self, a, scales, dtype=torch.bfloat16, out=None, stream=None):
        if dtype not in _DT_CODE:
            raise ValueError(f"mx.Linear: dtype {dtype}")
        return call(_native.mx_linear, stream, a, scales, self.w, self.w_scales, self.bias, self.K, self.N, self.bits,
                    _DT_CODE[dtype], out, not self.exact)
