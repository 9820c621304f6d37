"""int8 W8A8 linear: activations quantized per token inside the call, weights
held as int8 with one f32 scale an output channel.  The reference has no int8
activation path; the operator mirrors its quantized matmul (device buffers in,
device buffers out, stream last).  It has no gradient."""
import torch

from .native import _native, call
from .ops import _DT_CODE, _need_cuda

MAX_K = 132104  # where the int32 sum of K products stays exact


class Linear:
    """y = x @ (w * w_scale[:, None]).T + bias, with x rounded to int8 per row.

    w int8 [N, K], w_scale f32 [N], bias f32 [N] or None.  x is f32, f16 or
    bf16 [..., K] and y has its type.  A row's scale is amax / 127 (1 for a row
    of zeros), its codes round to even; a row that holds an infinity or a NaN
    gives NaN.  `out`, if given, does not overlap x.  K is padded once to a multiple of 128, so the weight is copied
    unless K is one already.
    """

    def __init__(self, w, w_scale, bias=None):
        _need_cuda(w, w_scale, bias)
        if w.dtype != torch.int8 or w.dim() != 2:
            raise ValueError("int8.Linear takes an int8 weight [N, K]")
        N, K = w.shape
        if not 0 < K <= MAX_K:
            raise ValueError(f"int8.Linear: K={K} (1..{MAX_K})")
        for name, t in (("w_scale", w_scale), ("bias", bias)):
            if t is not None and (t.shape != (N,) or t.dtype != torch.float32):
                raise ValueError(f"int8.Linear: {name} must be float32 [{N}]")
        ld = -(-K // 128) * 128
        if ld != K:
            packed = torch.zeros(N, ld, dtype=torch.int8, device=w.device)
            packed[:, :K] = w
        else:
            packed = w.contiguous()
            if packed.data_ptr() % 16:
                packed = packed.clone()
        self.N, self.K, self.ld = N, K, ld
        self.w, self.w_scale = packed, w_scale.contiguous()
        self.bias = None if bias is None else bias.contiguous()

    def forward(self, x, out=None, stream=None):
        return call(_native.linear, stream, x, self.w, self.w_scale, self.bias, self.K, out)

    __call__ = forward

    def codes(self, a, scales, dtype=torch.bfloat16, out=None, stream=None):
        """The same of activations that are in codes already: a int8 [..., K] (-127 .. 127),
        contiguous, and f32 scales [...], as norm.RmsNorm(...)(x, quant="int8") makes them; y is of dtype.
        Inputs that ask for a gradient, or have a tangent, are refused."""
        if dtype not in _DT_CODE:
            raise ValueError(f"int8.Linear: dtype {dtype}")
        if a.shape[-1:] != (self.K,):
            raise ValueError(f"int8.Linear: codes must be [..., {self.K}]")
        if self.ld != self.K:
            with torch.cuda.stream(stream):
                a = torch.nn.functional.pad(a, (0, self.ld - self.K))
        return call(_native.linear_codes, stream, a, scales, self.w, self.w_scale, self.bias, self.K,
                    _DT_CODE[dtype], out)
