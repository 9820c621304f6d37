"""int8 linear against its definition.

The codes, the int32 sum and the scales are exact, so the reference forms them
exactly (torch on the CPU, the sum in int64) and only the epilogue differs:
int32 to f32, two products and a sum, each 2^-24, then one rounding to the
output's type.
"""
import pytest
import torch

from ubridge_amd import int8

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(dev, M, K, N, dtype, bias, seed=0):
    g = torch.Generator().manual_seed(seed + M + K + N)
    x = (torch.randn(M, K, generator=g) * torch.exp(0.5 * torch.randn(K, generator=g))).to(dtype)
    w = torch.randint(-128, 128, (N, K), generator=g).to(torch.int8)
    ws = torch.rand(N, generator=g) * 2e-3 + 1e-4
    b = torch.randn(N, generator=g) if bias else None
    return x, w, ws, b, int8.Linear(w.to(dev), ws.to(dev), None if b is None else b.to(dev))


def want(x, w, ws, b, dev):
    """(value, size of the f32 errors) in 64 bits, from exact codes and scales."""
    xf = x.float().cpu()
    amax = xf.abs().amax(1)
    s = torch.where(amax > 0, amax / 127.0, torch.ones(()))
    q = torch.round(xf / s[:, None]).clamp(-127, 127)
    # sums of whole numbers below 2^31: exact in 64 bits
    dot = (q.double().to(dev) @ w.double().to(dev).t().contiguous()).cpu()
    y = dot * s.double()[:, None] * ws.double()
    size = y.abs()
    if b is not None:
        y, size = y + b.double(), size + b.double().abs()
    return y, size


def near(got, x, w, ws, b, dev):
    y, size = want(x, w, ws, b, dev)
    half = torch.finfo(got.dtype).eps / 2
    tol = half * y.abs() + (1 + half) * 2.0**-21 * size + torch.finfo(got.dtype).smallest_normal * half
    # values from half a step past the type's largest on round to infinity
    top = torch.finfo(got.dtype).max * (1 + half / 2)
    y = torch.where(y.abs() >= top, torch.full_like(y, torch.inf).copysign(y), y)
    tol = torch.where(y.isinf(), torch.zeros_like(y), tol)
    g = got.double().cpu()
    err = torch.where(g == y, torch.zeros_like(y), (g - y).abs())
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,bias", [
    (1, 1, 1, True), (1, 128, 128, False), (3, 131, 17, True), (2, 4096, 384, False), (5, 127, 8, True),
    (8, 640, 1000, False), (15, 256, 300, True), (16, 2048, 512, True), (17, 513, 257, True),
    (31, 384, 64, False), (33, 1000, 129, True), (64, 1024, 512, False), (100, 257, 1001, True),
    (129, 128, 255, True), (200, 704, 900, False), (256, 1024, 1024, True), (300, 3520, 257, False),
    (513, 129, 511, True), (1000, 320, 770, True)])
def test_linear(dev, dtype, M, K, N, bias):
    x, w, ws, b, lin = make(dev, M, K, N, dtype, bias)
    guard = torch.full((M + 1, N), 3.0, device=dev, dtype=dtype)
    near(lin(x.to(dev), out=guard[:M]), x, w, ws, b, dev)
    assert bool((guard[M] == 3.0).all())


@pytest.mark.parametrize("M,K,N", [(1, 14336, 4096), (16, 14336, 1024), (4, 8192, 9001), (2048, 1024, 1536),
                                   (1500, 4100, 2000), (16, 28672, 320), (640, 8192, 640)])
def test_linear_large(dev, M, K, N):
    x, w, ws, b, lin = make(dev, M, K, N, torch.bfloat16, True)
    near(lin(x.to(dev)), x, w, ws, b, dev)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,bias", [(40, 13970, 450, True), (490, 9272, 361, False), (114, 12604, 2482, True),
                                        (17, 20000, 33, False), (130, 5000, 129, True)])
def test_linear_parts(dev, dtype, M, K, N, bias):
    # long rows over few tiles: K in parts, some of unequal length
    x, w, ws, b, lin = make(dev, M, K, N, dtype, bias)
    y = lin(x.to(dev))
    near(y, x, w, ws, b, dev)
    assert torch.equal(y, lin(x.to(dev)))


@pytest.mark.parametrize("M", [1, 16, 70])
def test_extremes(dev, M):
    # the largest sum: every product -128 * 127, at the longest row
    K = int8.MAX_K
    w = torch.full((5, K), -128, dtype=torch.int8, device=dev)
    lin = int8.Linear(w, torch.ones(5, device=dev))
    x = torch.full((M, K), 127.0, device=dev)
    assert bool((lin(x) == -float(K * 127 * 128)).all())
    assert bool((lin(-x) == float(K * 127 * 128)).all())


def test_rows(dev):
    # zeros, infinities, NaN, denormals, ties and a row much smaller than its neighbour
    x, w, ws, b, lin = make(dev, 8, 640, 320, torch.float32, True)
    x[0] = 0.0
    x[1, 5] = float("inf")
    x[2, 639] = float("nan")
    x[3] *= 1e-30
    x[4] = torch.arange(640) % 255 - 127.0  # scale 1
    x[4, ::3] += 0.5
    x[4, 0], x[4, 1] = 127.0, -127.0
    x[5] = 1e-44  # scale 0: rounded off
    x[6] = 3e38
    y = lin(x.to(dev)).cpu()
    assert bool(y[1].isnan().all() and y[2].isnan().all())
    assert torch.equal(y[0], b)
    near(y[[3, 4, 6, 7]], x[[3, 4, 6, 7]], w, ws, b, dev)
    assert bool(torch.isfinite(y[5]).all())
    # the same rows in one type of 16 bits
    xb = x.bfloat16()
    yb = lin(xb.to(dev)).cpu()
    assert bool(yb[1].isnan().all() and yb[2].isnan().all())
    near(yb[[0, 3, 4, 6, 7]], xb[[0, 3, 4, 6, 7]], w, ws, b, dev)


def test_shapes_and_strides(dev):
    x, w, ws, b, lin = make(dev, 24, 200, 100, torch.bfloat16, True)
    y = lin(x.to(dev))
    assert torch.equal(lin(x.to(dev).view(2, 3, 4, 200)), y.view(2, 3, 4, 100))
    assert torch.equal(lin(x.to(dev)[0]), lin(x.to(dev)[:1])[0])
    wide = torch.zeros(24, 407, dtype=torch.bfloat16, device=dev)
    wide[:, 3:203] = x.to(dev)
    assert torch.equal(lin(wide[:, 3:203]), y)
    odd = torch.empty(24 * 200 + 1, dtype=torch.bfloat16, device=dev)[1:].view(24, 200)  # 2-byte aligned
    assert torch.equal(lin(odd.copy_(x)), y)
    assert lin(x.to(dev)[:0]).shape == (0, 100)
    # a weight that is a view: every other row of another
    lin2 = int8.Linear(torch.stack([w, w], 1).to(dev)[:, 0], ws.to(dev), b.to(dev))
    assert torch.equal(lin2(x.to(dev)), y)
    big = torch.zeros(100 * 256 + 1, dtype=torch.int8, device=dev)[1:].view(100, 256)
    big[:, :200] = w.to(dev)
    lin3 = int8.Linear(big, ws.to(dev), b.to(dev))
    assert torch.equal(lin3(torch.nn.functional.pad(x, (0, 56)).to(dev)), y)


@pytest.mark.parametrize("M", [1, 8, 40, 300])
def test_stream_and_graph(dev, M):
    x, w, ws, b, lin = make(dev, M, 512, 768, torch.bfloat16, True)
    x = x.to(dev)
    y = lin(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    z = lin(x, stream=side)
    side.synchronize()
    assert torch.equal(y, z)
    out = torch.empty_like(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lin(x, out=out)
    for i in range(4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, lin(x))


def test_refusals(dev):
    w = torch.zeros(16, 32, dtype=torch.int8, device=dev)
    s = torch.ones(16, device=dev)
    for args in ((w.float(), s), (w[0], s), (w, s[:3]), (w, s.half()), (w, s, s[:1]), (w.cpu(), s),
                 (torch.zeros(1, int8.MAX_K + 1, dtype=torch.int8, device=dev), s[:1]), (w[:, :0], s)):
        with pytest.raises(ValueError):
            int8.Linear(*args)
    lin = int8.Linear(w, s)
    x = torch.zeros(4, 32, device=dev)
    for bad in (x[:, :31], x.double(), x.cpu(), x.sum()):
        with pytest.raises(ValueError):
            lin(bad)
    for out in (torch.zeros(4, 15, device=dev), torch.zeros(4, 16, device=dev).half(),
                torch.zeros(16, 4, device=dev).t()):
        with pytest.raises(ValueError):
            lin(x, out=out)


def test_result_over_its_input_is_refused(dev):
    lin = int8.Linear(torch.ones(32, 32, dtype=torch.int8, device=dev), torch.ones(32, device=dev))
    pool = torch.ones(12, 32, device=dev)
    for out in (pool[:4], pool[3:7]):
        with pytest.raises(ValueError, match="overlaps"):
            lin(pool[:4], out=out)
    want = lin(pool[:4])
    lin(pool[:4], out=pool[4:8])
    assert torch.equal(pool[4:8], want)


def test_replaced_weights_are_checked(dev):
    x = torch.ones(4, 32, device=dev)
    for name, t in (("w", torch.ones(32, 16, dtype=torch.int8, device=dev)), ("w", torch.ones(32, 128, device=dev)),
                    ("w_scale", torch.ones(31, device=dev)), ("bias", torch.ones(32, device=dev).half())):
        lin = int8.Linear(torch.ones(32, 32, dtype=torch.int8, device=dev), torch.ones(32, device=dev))
        setattr(lin, name, t)
        with pytest.raises(ValueError):
            lin(x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(8, 8192, 40), (9, 8192, 40), (16, 4096, 100), (16, 4097, 100), (5, 13107, 33),
                                   (6, 13107, 33), (1, 65536, 17), (1, 65537, 17), (2, 32768, 50), (1, 132104, 5)])
def test_few_tokens_of_long_rows(dev, dtype, M, K, N):
    x, w, ws, b, lin = make(dev, M, K, N, dtype, True)
    near(lin(x.to(dev)), x, w, ws, b, dev)
