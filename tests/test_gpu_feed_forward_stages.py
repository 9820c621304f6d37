"""The dense half with activations in 4- and 8-bit blocks, from the norm to its result,
each stage against 64 bits from what the stage before it gave; and norms of many short
rows (heads), with their gradients."""
import pytest
import torch

from test_gpu_feed_forward import example, in_blocks, normed
from test_gpu_mx_sums import near as sums_near
from test_gpu_norm import EPS, gradients_hold, make, near, plain
from ubridge_amd import moe, mx, norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["fp4", "fp8"])
@pytest.mark.parametrize("tokens,hidden,inner", [(1, 192, 96), (7, 200, 97), (16, 1024, 512), (40, 320, 160), (300, 512, 384)])
def test_dense_half(dev, tokens, hidden, inner, act):
    g = torch.Generator().manual_seed(tokens)
    w13, w2, x, r = (torch.randn(*s, generator=g).bfloat16().to(dev) * c for s, c in (
        ((2 * inner, hidden), hidden**-0.5), ((hidden, inner), inner**-0.5), ((tokens, hidden), 1.0), ((tokens, hidden), 1.0)))
    n = norm.RmsNorm((1 + 0.1 * torch.randn(hidden, generator=g)).bfloat16().to(dev))
    h = (x.float() + r.float()).bfloat16()
    half = example.Dense(w13, w2, act)
    y, s = half(n, x, r)
    assert torch.equal(s, h)
    # the blocks: where a code is another one, the f32 value lay beside the border (3 * 2^-24)
    q = n(h, quant=act)
    got, want = mx.dequantize(*q, hidden, torch.float32).double(), normed(n, h)
    wide = torch.where(got == in_blocks(want, act), got, torch.maximum(in_blocks(want * (1 - 2.0**-22), act),
                                                                       in_blocks(want * (1 + 2.0**-22), act)))
    thin = torch.minimum(in_blocks(want * (1 - 2.0**-22), act), in_blocks(want * (1 + 2.0**-22), act))
    assert bool(((got == in_blocks(want, act)) | ((got <= wide) & (got >= thin))).all())

    def product(a, w, k, result):
        w = in_blocks(w, "fp4")
        sums_near(result, a @ w.t().contiguous(), a.abs() @ w.abs().t().contiguous(), k)
    gate_up = half.w13.codes(*q, torch.bfloat16)
    product(got, w13, hidden, gate_up)
    a = moe.silu_and_mul(gate_up)
    ga, up = gate_up.double().chunk(2, 1)
    want = torch.nn.functional.silu(ga) * up
    assert bool(((a.double() - want).abs() <= 3 * 2.0**-8 * want.abs() + 1e-30).all())
    out = half.w2(a)
    product(in_blocks(a, act), w2, inner, out)
    assert torch.equal(y, out)


@pytest.mark.parametrize("R,C,dtype", [(65536, 128, torch.bfloat16), (65536, 64, torch.float16), (30000, 80, torch.bfloat16),
                                       (20011, 96, torch.float32), (9000, 256, torch.bfloat16), (70000, 33, torch.float16),
                                       (100000, 1, torch.float32), (4100, 511, torch.bfloat16)])
@pytest.mark.parametrize("residual", [True, False])
def test_many_short_rows(dev, R, C, dtype, residual):
    x, res, w = make(dev, R, C, dtype, torch.float32 if C % 2 else dtype, residual)
    h, y = plain(x, res, w)
    got = norm.RmsNorm(w, EPS)(x, res)
    near(got[0] if residual else got, y)
    if residual:
        assert torch.equal(got[1], h)
    gradients_hold(dev, R, C, dtype, residual)
