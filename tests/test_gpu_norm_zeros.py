"""Zeros among the normed values keep their sign in e4m3 codes, as in blocks and in
fp8.quantize_rows of the f32 result."""
import pytest
import torch

from ubridge_amd import fp8, norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("R,C", [(3, 64), (5, 1000), (2000, 96), (40, 9001)])
@pytest.mark.parametrize("gain", [1.0, 2.0**100])  # (a scale past 2^60 is divided by)
def test_signs(dev, R, C, dtype, gain):
    g = torch.Generator().manual_seed(R)
    x = torch.randn(R, C, generator=g)
    x[torch.rand(R, C, generator=g) < 0.3] = 0.0
    x[torch.rand(R, C, generator=g) < 0.3] = -0.0
    x = x.to(dtype).to(dev)
    w = (torch.randn(C, generator=g) * gain).to(dev)
    w[::7] = 0.0
    n = norm.RmsNorm(w, 1e-6)
    q, s = n(x, quant="e4m3")
    # the sign of h r w, r > 0, also of zeros
    want = torch.signbit(x.float()) ^ torch.signbit(w)
    assert torch.equal(q.view(torch.uint8) >= 128, want)
    if dtype == torch.float32 and C % 16 == 0 and gain == 1.0:
        same, scale = fp8.quantize_rows(n(x))
        assert torch.equal(scale.flatten(), s) and torch.equal(same.view(torch.uint8), q)
    codes, _ = n(x, quant="fp8")
    assert torch.equal(codes[:, :C] >= 128, want)
    codes, _ = n(x, quant="fp4")
    i = torch.stack([codes & 8, codes >> 4 & 8], -1).flatten(1)[:, :C]
    assert torch.equal(i > 0, want)
