"""Results written into a caller's tensor raise its version, so that a graph that saved
its old values refuses to run backward over the new ones."""
import pytest
import torch

from ubridge_amd import attention, int8, mx, norm

pytestmark = pytest.mark.gpu


def saved(t):
    """A result whose backward needs t's present values."""
    w = torch.ones_like(t, requires_grad=True)
    return (w * t).sum(), w


def refuses(loss):
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def rand(dev, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(len(shape))).bfloat16().to(dev)


@pytest.mark.parametrize("how", ["no_grad", "detach"])
def test_a_norm_over_what_a_norm_saved(dev, how):
    # h of the first is what its backward starts from
    x, res, a = (rand(dev, 6, 200) for _ in range(3))
    n = norm.RmsNorm(torch.ones(200, device=dev, requires_grad=True))
    m = norm.RmsNorm(torch.ones(200, device=dev))
    y, h = n(x, res)
    if how == "no_grad":
        with torch.no_grad():
            m(a, h, residual_out=h)
    else:
        m(a, h.detach(), residual_out=h.detach())
    refuses(y.float().sum())
    y, h = n(x, res)  # and left alone it runs
    y.float().sum().backward()


@pytest.mark.parametrize("quant", [None, "int8", "fp4"])
def test_residual_out(dev, quant):
    x, r = rand(dev, 6, 200), rand(dev, 6, 200)
    n = norm.RmsNorm(torch.ones(200, device=dev))
    loss, _ = saved(r)
    v = r._version
    n(x, r, quant=quant)
    assert r._version == v  # read only
    n(x, r, quant=quant, residual_out=r)
    assert r._version > v
    refuses(loss)
    v = x._version
    n(x, r, quant=quant, residual_out=x[:])  # (a view's base is the same memory)
    assert x._version > v
    with torch.inference_mode():
        r = rand(dev, 6, 200)
        n(x.clone(), r, residual_out=r)


def outs(dev):
    """(call(out), result's shape) of each linear"""
    x = rand(dev, 5, 256)
    w = torch.randint(-127, 128, (48, 256), dtype=torch.int8, device=dev)
    i8 = int8.Linear(w, torch.ones(48, device=dev))
    m = mx.Linear(*mx.quantize(rand(dev, 48, 256)), 256)
    codes = mx.quantize(x, "fp4")
    q = torch.randint(-127, 128, (5, 256), dtype=torch.int8, device=dev)
    s = torch.ones(5, device=dev)
    qkv = rand(dev, 2, 4, 64), rand(dev, 8, 2, 16, 64), rand(dev, 8, 2, 16, 64)
    tables = torch.arange(4, device=dev, dtype=torch.int32).view(2, 2)
    lens = torch.tensor([20, 7], device=dev, dtype=torch.int32)
    return {"int8": (lambda o: i8(x, out=o), (5, 48)), "int8 codes": (lambda o: i8.codes(q, s, out=o), (5, 48)),
            "mx": (lambda o: m(x, out=o), (5, 48)), "mx codes": (lambda o: m.codes(*codes, out=o), (5, 48)),
            "decode": (lambda o: attention.paged_decode(*qkv, tables, lens, out=o), (2, 4, 64))}


@pytest.mark.parametrize("name", ["int8", "int8 codes", "mx", "mx codes", "decode"])
def test_out(dev, name):
    call, shape = outs(dev)[name]
    out = torch.zeros(shape, device=dev, dtype=torch.bfloat16)
    loss, _ = saved(out)
    call(out)
    refuses(loss)
    with torch.inference_mode():
        call(torch.zeros(shape, device=dev, dtype=torch.bfloat16))


def test_results_that_ask_for_a_gradient(dev):
    x, r = rand(dev, 6, 200), rand(dev, 6, 200)
    n = norm.RmsNorm(torch.ones(200, device=dev))
    leaf = torch.zeros(6, 200, device=dev, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        n(x, r, residual_out=leaf)
    with torch.no_grad():
        n(x, r, residual_out=leaf)
    assert torch.equal(leaf.detach(), (x.float() + r.float()).bfloat16())
    for name in ("int8 codes", "mx", "mx codes"):
        call, shape = outs(dev)[name]
        leaf = torch.zeros(shape, device=dev, dtype=torch.bfloat16, requires_grad=True)
        with pytest.raises(ValueError, match="no gradient"):
            call(leaf)
        with torch.no_grad():
            call(leaf)
