"""Root-mean-square norm against its definition in 64 bits.

The residual's sum is f32, rounded to the type: exactly repeated here.  y is three
f32 operations from exact values (r, rounded once from 64 bits; h r; times w): 3 *
2^-24, below 2^-22 of it, then one rounding to what goes out.
"""
import math

import pytest
import torch

from ubridge_amd import fp8, int8, mx, norm
from ubridge_amd.native import _native

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
EPS = 1e-6
F32 = 2.0**-22  # of y


def make(dev, R, C, dtype, wdtype=None, residual=True, seed=0):
    g = torch.Generator().manual_seed(seed + R + C)
    x = (torch.randn(R, C, generator=g) * torch.exp(0.5 * torch.randn(C, generator=g))).to(dtype)
    res = torch.randn(R, C, generator=g).to(dtype) if residual else None
    w = (1 + 0.3 * torch.randn(C, generator=g)).to(wdtype or dtype)
    return x.to(dev), None if res is None else res.to(dev), w.to(dev)


def plain(x, res, w, eps=EPS):
    """(h, y in 64 bits)"""
    h = x if res is None else (x.float() + res.float()).to(x.dtype)
    d = h.double()
    return h, d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps) * w.double()


def near(got, y, rel=F32):
    half = torch.finfo(got.dtype).eps / 2
    tol = (half + rel * (1 + half)) * y.abs() + torch.finfo(got.dtype).smallest_normal * half
    err = (got.double() - y).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


SHAPES = [(1, 1), (1, 64), (3, 7), (2, 8), (5, 100), (8, 4096), (1, 5003), (33, 513), (7, 2048), (1024, 64), (1030, 519),
          (1027, 1000), (600, 4100), (513, 8192), (4, 9000), (2, 16384), (1500, 33)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,C", SHAPES)
@pytest.mark.parametrize("residual", [True, False])
def test_norm(dev, R, C, dtype, residual):
    wd = torch.float32 if C % 2 else dtype
    x, res, w = make(dev, R, C, dtype, wd, residual)
    h, y = plain(x, res, w)
    got = norm.RmsNorm(w, EPS)(x, res)
    if residual:
        got, gh = got
        assert torch.equal(gh, h)
    near(got, y)


@pytest.mark.parametrize("dtype,C", [(torch.bfloat16, 32768), (torch.float16, 20001), (torch.float32, 16384)])
def test_long_rows(dev, dtype, C):
    x, res, w = make(dev, 3, C, dtype)
    h, y = plain(x, res, w)
    got, gh = norm.RmsNorm(w, EPS)(x, res)
    assert torch.equal(gh, h)
    near(got, y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,C", SHAPES + [(2, 32)])
@pytest.mark.parametrize("quant", ["int8", "e4m3"])
def test_codes(dev, R, C, dtype, quant):
    x, res, w = make(dev, R, C, dtype)
    h, y = plain(x, res, w)
    q, s, gh = norm.RmsNorm(w, EPS)(x, res, quant=quant)
    assert torch.equal(gh, h)
    most = 127.0 if quant == "int8" else 448.0
    amax = y.abs().amax(1)
    want = torch.where(amax > 0, amax / most, torch.ones_like(amax))
    near(s, want, F32 + 2.0**-24)
    v = q if quant == "int8" else q.view(torch.float8_e4m3fn)
    v = v.double() * s.double()[:, None]
    # off by half a step of the code, and the f32 errors of y and of the quotient (2^-24)
    step = s.double()[:, None] if quant == "int8" else torch.maximum(y.abs() * 2.0**-3, s.double()[:, None] * 2.0**-9)
    assert bool(((v - y).abs() <= step / 2 * (1 + 2.0**-20) + y.abs() * 2 * F32).all())


@pytest.mark.parametrize("R,C", [(3, 7), (8, 4096), (1030, 519), (600, 1000), (5, 9001)])
def test_codes_are_of_the_f32_result(dev, R, C):
    # of f32 rows the result itself is there: codes and blocks are its, bit for bit
    x, _, w = make(dev, R, C, torch.float32, residual=False)
    n = norm.RmsNorm(w, EPS)
    y = n(x)
    q, s = n(x, quant="int8")
    # (quotients on the CPU: torch's on the device multiply by a number's inverse)
    yc, sc = y.cpu(), s.cpu()
    amax = yc.abs().amax(1)
    assert torch.equal(sc, torch.where(amax > 0, amax / 127.0, torch.ones_like(amax)))
    assert torch.equal(q.cpu(), torch.round(yc / sc[:, None]).clamp(-127, 127).to(torch.int8))
    q, s = n(x, quant="e4m3")
    want = fp8.quantize_rows(y)
    assert torch.equal(q, want[0]) and torch.equal(s, want[1])
    for fmt in ("fp4", "fp8"):
        got, want = n(x, quant=fmt), mx.quantize(y, fmt)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("R,C", [(1, 1), (3, 33), (8, 4096), (1100, 200), (600, 4100), (2, 20000)])
def test_blocks(dev, R, C, dtype, fmt):
    # the f32 result of the same values: that of f32 rows (r may differ by its last bit,
    # were the 64-bit sums of another order to lie on both sides of a border: not here)
    x, res, w = make(dev, R, C, dtype, torch.float32)
    q, s, h = norm.RmsNorm(w, EPS)(x, res, quant=fmt)
    if C <= 16384:
        want = mx.quantize(norm.RmsNorm(w, EPS)(h.float()), fmt)
        assert torch.equal(q, want[0]) and torch.equal(s, want[1])
    _, y = plain(x, res, w)
    v = mx.dequantize(q, s, C, torch.float32).double()
    unit = torch.exp2(s.double() - 127).repeat_interleave(32, 1)[:, :C]
    # steps within a block: a quarter of the binade (e4m3: a sixteenth), and the clipped top
    big = unit * (2 if fmt == "fp4" else 64)
    assert bool(((v - y).abs() <= big * (1 + 2.0**-20)).all())
    assert bool((q.view(R, -1)[:, -(-C // 2 if fmt == "fp4" else -C):] == 0).all())


def test_scales_of_extreme_rows(dev):
    x = torch.zeros(6, 256, device=dev)
    x[1, 3] = 3e38  # squares that f32 does not hold
    x[2] = 1e-30
    x[3] = 1e30
    x[4, 5] = math.inf
    x[5, 7] = math.nan
    w = torch.ones(256, device=dev)
    n = norm.RmsNorm(w, 0.0)
    y = n(x[1:4])
    assert torch.equal(y[1], torch.ones_like(y[1])) and torch.equal(y[2], torch.ones_like(y[2]))
    assert float(y[0, 3]) == 16.0 and int((y[0] != 0).sum()) == 1
    n = norm.RmsNorm(w, EPS)
    assert bool((n(x[:1]) == 0).all())
    for quant in ("int8", "e4m3"):
        q, s = n(x, quant=quant)
        assert float(s[0]) == 1 and bool((q[0] == 0).all())
        assert bool(torch.isnan(s[4:]).all()) and bool((q[4:] == 0).all())
        assert bool(torch.isfinite(s[:4]).all())
    q, s = n(x, quant="fp8")
    assert int(s[4, 0]) == 255 and int(s[5, 0]) == 255 and bool((s[5] == 255).all())


@pytest.mark.parametrize("gain", [2.0**-100, 2.0**-62, 2.0**-57, 2.0**55, 2.0**60, 2.0**100])
@pytest.mark.parametrize("C", [200, 5003])
def test_codes_at_extreme_scales(dev, C, gain):
    # the result's own quotients, bit for bit, also where residuals of a division would
    # underflow (the gains' own spread puts scales on both sides of 2^-60 and 2^60)
    x, _, w = make(dev, 9, C, torch.float32, residual=False)
    n = norm.RmsNorm(w * gain, EPS)
    y = n(x * torch.exp2(torch.arange(9.0, device=dev) - 4)[:, None])
    q, s = n(x * torch.exp2(torch.arange(9.0, device=dev) - 4)[:, None], quant="int8")
    yc, sc = y.cpu(), s.cpu()
    assert torch.equal(sc, yc.abs().amax(1) / 127.0)
    assert torch.equal(q.cpu(), torch.round(yc / sc[:, None]).clamp(-127, 127).to(torch.int8))
    q, s = n(x * torch.exp2(torch.arange(9.0, device=dev) - 4)[:, None], quant="e4m3")
    sc = s.cpu()
    assert torch.equal(sc, yc.abs().amax(1) / 448.0)
    want = (yc / sc[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(q.cpu().view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES)
def test_in_place_strides_and_shapes(dev, dtype):
    x, res, w = make(dev, 24, 520, dtype)
    n = norm.RmsNorm(w, EPS)
    y, h = n(x, res)
    r2 = res.clone()
    y2, h2 = n(x, r2, residual_out=r2)
    assert h2.data_ptr() == r2.data_ptr() and torch.equal(h2, h) and torch.equal(y2, y)
    x2 = x.clone()
    y2, h2 = n(x2, res, residual_out=x2)
    assert torch.equal(x2, h) and torch.equal(y2, y)
    wide = torch.cat([x, x], 1)[:, :520]
    assert not wide.is_contiguous() and torch.equal(n(wide, res)[0], y)
    y3, h3 = n(x.view(2, 3, 4, 520), res.view(2, 3, 4, 520))
    assert torch.equal(y3.view(24, 520), y) and y3.shape == (2, 3, 4, 520)
    q, s, _ = n(x.view(2, 12, 520), res.view(2, 12, 520), quant="int8")
    assert q.shape == (2, 12, 520) and s.shape == (2, 12)
    assert torch.equal(n(x[0], res[0])[0], y[0])
    e = n(x[:0], res[:0])
    assert e[0].shape == (0, 520)
    # rows that start at any element
    odd = torch.empty(24 * 520 + 1, device=dev, dtype=dtype)[1:].view(24, 520).copy_(x)
    assert torch.equal(n(odd, res)[0], y)


def test_refusals(dev):
    x, res, w = make(dev, 4, 64, torch.bfloat16)
    n = norm.RmsNorm(w)
    for call in (lambda: n(x.double()), lambda: n(x.cpu()), lambda: n(x[:, :32]), lambda: n(x, res[:2]), lambda: n(x, res.float()),
                 lambda: n(x, quant="int4"), lambda: n(x, residual_out=res), lambda: n(x, res, residual_out=res.t().contiguous().t()),
                 lambda: norm.RmsNorm(w.half())(x), lambda: norm.RmsNorm(w, -1.0)(x),
                 lambda: norm.RmsNorm(torch.ones(40000, device=dev))(torch.ones(2, 40000, device=dev)),
                 lambda: n(x.clone().requires_grad_(), quant="int8"),
                 lambda: n(x.clone().requires_grad_(), res, residual_out=res)):
        with pytest.raises(ValueError):
            call()
    big = torch.zeros(5, 64, device=dev, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="in part"):
        n(big[:4], big[:4].clone(), residual_out=big[1:])
    with torch.no_grad():
        n(x.clone().requires_grad_(), quant="int8")


# ---------------------------------------------------------------- gradients
def gradients(x, res, w, dy, dh):
    """The formula's in 64 bits, and the sizes that its f32 errors scale with."""
    h, _ = plain(x, res, w)
    h, wd, dy = h.double(), w.double(), dy.double()
    C = h.shape[1]
    r = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
    g = dy * wd
    m = r * r * (g * h).sum(1, keepdim=True) / C
    dx = r * (g - h * m)
    size = r * (g.abs() + h.abs() * r * r * (g * h).abs().sum(1, keepdim=True) / C)
    if dh is not None:
        dx, size = dx + dh.double(), size + dh.double().abs()
    return dx, size, (dy * h * r).sum(0), (dy * h * r).abs().sum(0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,C", [(1, 1), (1, 64), (3, 7), (5, 513), (8, 4096), (600, 1000), (1500, 72), (700, 4100),
                                 (40, 8200), (3, 16384)])
@pytest.mark.parametrize("residual", [True, False])
def test_gradients(dev, R, C, dtype, residual):
    gradients_hold(dev, R, C, dtype, residual)


@pytest.mark.parametrize("dtype,C", [(torch.bfloat16, 32768), (torch.float16, 20001), (torch.bfloat16, 16392), (torch.float32, 8196)])
@pytest.mark.parametrize("residual", [True, False])
def test_gradients_of_long_rows(dev, C, dtype, residual):
    gradients_hold(dev, 600, C, dtype, residual)


def gradients_hold(dev, R, C, dtype, residual):
    x, res, w = make(dev, R, C, dtype, torch.float32 if C % 2 else dtype, residual)
    g = torch.Generator().manual_seed(R * C)
    dy = torch.randn(R, C, generator=g).to(dtype).to(dev)
    dh = torch.randn(R, C, generator=g).to(dtype).to(dev) if residual else None
    leaves = [t.requires_grad_() for t in (x, res, w) if t is not None]
    out = norm.RmsNorm(w, EPS)(x, res)
    y, h = out if residual else (out, None)
    got = torch.autograd.grad([y, h] if residual else [y], leaves, [dy, dh] if residual else [dy])
    dx, size, dw, wsize = gradients(x.detach(), None if res is None else res.detach(), w.detach(), dy, dh)
    half = torch.finfo(dtype).eps / 2
    # r, g, m, h m, the difference, times r, plus dh: 8 roundings of 2^-24 at most
    tol = half * dx.abs() + 2.0**-21 * size * (1 + half) + torch.finfo(dtype).smallest_normal * half
    for d in got[:-1]:
        assert d.dtype == dtype
        assert bool(((d.double() - dx).abs() <= tol).all())
    # rows of a workgroup, workgroups of a wavefront, wavefronts, and 3 roundings a term
    n = math.ceil(R / 512) + math.ceil(min(R, 512) / 16) + 16 + 3
    hw = torch.finfo(w.dtype).eps / 2
    assert bool(((got[-1].double() - dw).abs() <= hw * dw.abs() + (1 + hw) * n * 2.0**-24 * wsize).all())


def test_gradients_by_differences(dev):
    R, C = 6, 96
    x, res, w = make(dev, R, C, torch.float32)
    g = torch.Generator().manual_seed(5)
    vx, vr, vw = (torch.randn(s, generator=g).to(dev) for s in ((R, C), (R, C), (C,)))
    dy, dh = torch.randn(R, C, generator=g).to(dev), torch.randn(R, C, generator=g).to(dev)

    def f(t):
        y, h = norm.RmsNorm(w + t * vw, EPS)(x + t * vx, res + t * vr)
        return float((y.double() * dy).sum() + (h.double() * dh).sum())
    t = 2.0**-7
    diff = (f(t) - f(-t)) / (2 * t)
    leaves = [a.clone().requires_grad_() for a in (x, res, w)]
    y, h = norm.RmsNorm(leaves[2], EPS)(leaves[0], leaves[1])
    grads = torch.autograd.grad([y, h], leaves, [dy, dh])
    along = sum(float((a.double() * b).sum()) for a, b in zip(grads, (vx, vr, vw)))
    # f32 errors of both values, 2^-22 of R C terms of size about |y dy| each, over 2 t; and
    # the third derivative's t^2 / 6, below one term's size each
    terms = float((y.detach().double() * dy).abs().sum() + (h.detach().double() * dh).abs().sum())
    assert abs(diff - along) <= terms * (2 * 2.0**-22 / (2 * t) + t * t)


def test_gradient_paths(dev):
    x, res, w = make(dev, 9, 200, torch.float32)
    leaves = [t.requires_grad_() for t in (x, res, w)]
    n = norm.RmsNorm(w, EPS)
    y, h = n(x, res)
    # h alone: the identity, and nothing for the gain
    d = torch.autograd.grad(h.sum(), leaves, retain_graph=True)
    assert bool((d[0] == 1).all()) and bool((d[1] == 1).all()) and bool((d[2] == 0).all())
    # y alone, with an expanded gradient
    a = torch.autograd.grad(y.sum(), leaves, retain_graph=True)
    b = torch.autograd.grad([y, h], leaves, [torch.ones_like(y), torch.zeros_like(h)])
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    # one leaf
    y, h = n(x.detach(), res)
    c = torch.autograd.grad(y.sum(), [res])
    assert torch.equal(c[0], a[1])
    y = norm.RmsNorm(w, EPS)(x.detach())
    (dw,) = torch.autograd.grad(y.sum(), [w])
    assert dw.shape == w.shape
    # not twice
    y, h = n(x, res)
    (g,) = torch.autograd.grad(y.sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    # no rows
    e = torch.zeros(0, 200, device=dev, requires_grad=True)
    ge, gw = torch.autograd.grad(n(e).sum(), [e, w])
    assert ge.shape == (0, 200) and bool((gw == 0).all())
    # .grad of both leaves of one sum are tensors of their own
    y, h = n(x, res)
    (y * 2 + h).sum().backward()
    assert x.grad.data_ptr() != res.grad.data_ptr() and torch.equal(x.grad, res.grad)


def test_forward_mode_is_refused(dev):
    x, res, w = make(dev, 4, 64, torch.float32)
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: norm.RmsNorm(w, EPS)(d), lambda: norm.RmsNorm(w, EPS)(x, d), lambda: norm.RmsNorm(d[0], EPS)(x, quant="int8")):
            with pytest.raises(ValueError, match="forward mode"):
                call()
        near(norm.RmsNorm(w, EPS)(x), plain(x, None, w)[1])


def test_the_gradient_is_of_the_calls_stream(dev):
    # forward on a side stream that is busy, its backward asked for from another: it comes
    # after, without a wait of the caller's
    x, res, w = (t.requires_grad_() for t in make(dev, 64, 4096, torch.bfloat16))
    n = norm.RmsNorm(w, EPS)
    dy = torch.randn(64, 4096, device=dev).bfloat16()
    want = torch.autograd.grad(n(x, res), (x, res, w), (dy, dy))
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a = torch.ones(4096, 4096, device=dev)
            for _ in range(8):
                a = a.matmul(a).clamp(max=1)
        y, h = n(x, res, stream=side)
        got = torch.autograd.grad((y, h), (x, res, w), (dy, dy))
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        torch.cuda.current_stream().wait_stream(side)


def test_repeats_its_bits_and_streams(dev):
    x, res, w = make(dev, 1500, 1000, torch.bfloat16)
    w.requires_grad_()
    n = norm.RmsNorm(w, EPS)
    dy = torch.randn(1500, 1000, device=dev).bfloat16()

    def run(stream=None):
        y, h = n(x, res, stream=stream)
        return y, h, torch.autograd.grad(y, [w], dy)[0]
    want = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad():
        got = n(x, res, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("quant", [None, "int8", "e4m3", "fp4", "fp8"])
def test_graph(dev, quant):
    x, res, w = make(dev, 16, 1000, torch.bfloat16)
    n = norm.RmsNorm(w, EPS)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        n(x, res, quant=quant)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = n(x, res, quant=quant)
    for seed in range(3):
        a, b, _ = make(dev, 16, 1000, torch.bfloat16, seed=seed)
        x.copy_(a), res.copy_(b)
        want = n(x, res, quant=quant)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("M", [1, 16, 40])
@pytest.mark.parametrize("K", [512, 520])
def test_int8_linear_takes_the_codes(dev, M, K):
    # the linear's own rule on the same values gives the same codes, so the same result
    x, _, w = make(dev, M, K, torch.float32, residual=False)
    g = torch.Generator().manual_seed(1)
    wq = torch.randint(-127, 128, (96, K), generator=g, dtype=torch.int8).to(dev)
    lin = int8.Linear(wq, torch.rand(96, generator=g).to(dev), torch.randn(96, generator=g).to(dev))
    n = norm.RmsNorm(w, EPS)
    q, s = n(x, quant="int8")
    want = lin(n(x))
    got = lin.codes(q, s, torch.float32)
    assert torch.equal(got, want)
    out = torch.empty(M, 96, device=dev, dtype=torch.bfloat16)
    assert torch.equal(lin.codes(q, s, out=out), want.bfloat16())
    side = torch.cuda.Stream()
    for _ in range(5):  # all of the call is the stream's, a copy to padded rows too
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            late = torch.empty_like(q).fill_(0)
            torch.ones(4096, 4096, device=dev).matmul(torch.ones(4096, 4096, device=dev))
            late.copy_(q)
        got = lin.codes(late, s, torch.float32, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        late.record_stream(torch.cuda.current_stream())
    for call in (lambda: lin.codes(q.float(), s), lambda: lin.codes(q[:, :4], s), lambda: lin.codes(q, s[:0]),
                 lambda: lin.codes(q, s, torch.float64), lambda: lin.codes(q, s, torch.float32, out=out)):
        with pytest.raises(ValueError):
            call()


def test_fp8_gemm_takes_the_codes(dev):
    x, _, w = make(dev, 40, 512, torch.float32, residual=False)
    n = norm.RmsNorm(w, EPS)
    g = torch.Generator().manual_seed(1)
    wq, ws = fp8.quantize_rows(torch.randn(96, 512, generator=g).to(dev))
    q, s = n(x, quant="e4m3")
    want = fp8.gemm(*fp8.quantize_rows(n(x)), wq, ws)
    assert torch.equal(fp8.gemm(q, s, wq, ws), want)


def test_rows_past_32_bits(dev):
    # 2.3e9 elements: the last rows are those of a call of their own
    n = norm.RmsNorm(torch.rand(32768, device=dev), EPS)
    x = torch.empty(70000, 32768, device=dev, dtype=torch.bfloat16).normal_()
    y, h = n(x, x)
    want = n(x[-3:], x[-3:])
    assert torch.equal(y[-3:], want[0]) and torch.equal(h[-3:], want[1])
    del h
    leaf = x.requires_grad_()
    (dx,) = torch.autograd.grad(n(leaf), [leaf], y)
    last = x.detach()[-3:].clone().requires_grad_()
    (want,) = torch.autograd.grad(n(last), [last], y[-3:])
    assert torch.equal(dx[-3:], want)


def test_a_captured_gradient_refuses_leaves_of_a_living_eager_graph(dev):
    x, res, w = make(dev, 8, 256, torch.bfloat16)
    w.requires_grad_()
    n = norm.RmsNorm(w, EPS)
    y = n(x, res)[0]  # lives, on the default stream
    assert _native.default_stream_leaf(x, None, w) and not _native.default_stream_leaf(x, res)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="lives"):
            n(x, res)
        with torch.no_grad():
            z = n(x, res)[0]  # without a gradient: as ever
    graph.replay()
    assert torch.equal(z, y)
    del y
    assert not _native.default_stream_leaf(x, w)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = n(x, res)[0]
    assert not _native.default_stream_leaf(x, w)


def test_gradient_in_a_graph(dev):
    x, res, w = (t.requires_grad_() for t in make(dev, 40, 1000, torch.bfloat16))
    dy, dh = (torch.randn(40, 1000, device=dev).bfloat16() for _ in "yh")
    n = norm.RmsNorm(w, EPS)

    def run():
        y, h = n(x, res)
        return [y.detach(), h.detach(), *torch.autograd.grad([y, h], [x, res, w], [dy, dh])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for seed in range(3):
        with torch.no_grad():
            for t, v in zip((x, res, w), make(dev, 40, 1000, torch.bfloat16, seed=seed + 1)):
                t.copy_(v)
            dy.normal_(), dh.normal_()
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        want = run()
        assert all(torch.equal(a, b) for a, b in zip(kept, want))
