"""Root-mean-square norm of a residual stream: the addition to it, the norm, and
the rounding that the next product wants, in one launch; differentiable where the
result keeps its type."""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .native import _native, call
from .ops import _need_cuda
from .rope import _level, _stored

_OUT = {None: 0, "int8": 1, "e4m3": 2, "fp4": 3, "fp8": 4}


class RmsNorm:
    """y = h * weight / sqrt(mean(h ** 2) + eps), with h = x + residual rounded to
    x's type (h = x without a residual): the norm is of the stream as it is stored.

    weight [C] f32, or of x's type; x and residual [..., C] f32, f16 or bf16, a row
    at most 64 KiB.  norm(x) -> y; norm(x, residual) -> (y, h), h in `residual_out` if
    it is given, which may be residual or x itself.  quant rounds y from f32 for the
    next product and puts two tensors in its place:

      "int8"        codes int8 [..., C] and f32 scales [...], amax / 127 (1 for a row
                    of zeros), for int8.Linear.codes
      "e4m3"        codes uint8 and f32 scales, amax / 448, for fp8.gemm
      "fp4", "fp8"  microscaled blocks as mx.quantize makes them, for mx.Linear.codes

    A NaN makes its row NaN; an infinity is NaN in its place, and the rest of its row
    zeros.  Codes of such a row are 0 under a scale of NaN; of blocks, those that hold
    a NaN are NaN.  At most 2 ** 22 - 1 rows.  Without quant the call is differentiable, once,
    in x, residual and weight; with it, or into residual_out, it has no gradient and
    refuses inputs, or a residual_out, that ask for one; inputs with a tangent (forward
    mode) are always refused.  residual_out's version rises, as after any write in place.  A call that
    is captured for its gradient is refused while results of an eager one of the same
    leaves live that was on the default stream.
    """

    def __init__(self, weight, eps=1e-6):
        _need_cuda(weight)
        self.weight, self.eps = weight, float(eps)

    def forward(self, x, residual=None, quant=None, residual_out=None, stream=None):
        if quant not in _OUT:
            raise ValueError(f"RmsNorm: quant {quant!r} (one of {list(_OUT)})")
        if _level() >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                 for t in (x, residual, self.weight)):
            raise ValueError("RmsNorm: no forward mode")
        r = call(_native.norm, stream, x, self.weight, residual, residual_out, self.eps, _OUT[quant])
        if r is None:  # a gradient is asked for
            with torch.cuda.stream(stream):  # the backward pass is of the same stream
                if torch.cuda.is_current_stream_capturing() and _native.default_stream_leaf(x, residual, self.weight):
                    raise ValueError("RmsNorm: captured with a gradient while an eager graph of the same leaves lives: "
                                     "delete its results first, or make them on another stream than the default one")
                y, h = _Norm.apply(x, residual, self.weight, self.eps)
            return y if residual is None else (y, h)
        return r

    __call__ = forward


class _Norm(torch.autograd.Function):
    """(y, h).  The gradient starts from h as it is stored; of x and of residual it
    is the same."""

    @staticmethod
    def forward(ctx, x, residual, w, eps):
        r = call(_native.norm, None, x, w, residual, None, eps, 0)
        y, h = (r, None) if residual is None else r
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x if h is None else h, w)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        h, w = ctx.saved_tensors
        need_x, need_res, need_w = ctx.needs_input_grad[:3]
        if dy is None:  # only h was used
            dx, dw = dh, torch.zeros_like(w) if need_w else None
        else:
            dx, dw = call(_native.norm_grad, None, h.contiguous(), w, _stored(dy), _stored(dh), ctx.eps,
                          need_x or need_res, need_w)
        return dx if need_x else None, dx if need_res else None, dw, None
