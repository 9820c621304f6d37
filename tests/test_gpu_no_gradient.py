"""Operators without a gradient refuse inputs that ask for one, or that have a tangent:
a result without it would cut the graph silently."""
import pytest
import torch
from torch.autograd import forward_ad

from ubridge_amd import int8, moe, mx

pytestmark = pytest.mark.gpu


def calls(dev):
    """name: (call, its floating inputs)"""
    g = torch.Generator().manual_seed(0)

    def rand(*shape):
        return torch.randn(*shape, generator=g).bfloat16().to(dev)
    x, b = rand(5, 256), torch.randn(48, generator=g).to(dev)
    wq = torch.randint(-127, 128, (48, 256), generator=g, dtype=torch.int8).to(dev)
    q = torch.randint(-127, 128, (5, 256), generator=g, dtype=torch.int8).to(dev)
    blocks = mx.quantize(rand(48, 256))
    experts = [torch.randint(-127, 128, s, generator=g, dtype=torch.int8).to(dev) for s in ((8, 64, 256), (8, 256, 32))]
    return {
        "quantize": (lambda x: mx.quantize(x)[0], [x]),
        "mx.Linear": (lambda x, b: mx.Linear(*blocks, 256, bias=b)(x), [x, b]),
        "mx.Linear.codes": (lambda b: mx.Linear(*blocks, 256, bias=b).codes(*mx.quantize(x)), [b]),
        "int8.Linear.codes": (lambda s, ws, b: int8.Linear(wq, ws, b).codes(q, s),
                              [torch.rand(5, generator=g).to(dev), torch.rand(48, generator=g).to(dev), b]),
        "decode": (lambda x, lg, w13, w2: moe.FusedMoE(w13, w2, topk=2).decode(x, lg),
                   [x, rand(5, 8), rand(8, 64, 256), rand(8, 256, 32)]),
        "decode int8": (lambda x, lg, s13, s2: moe.FusedMoE(*experts, s13, s2, topk=2).decode(x, lg),
                        [x, rand(5, 8).float(), rand(8, 64), rand(8, 256)]),
    }


NAMES = ["quantize", "mx.Linear", "mx.Linear.codes", "int8.Linear.codes", "decode", "decode int8"]


@pytest.mark.parametrize("name", NAMES)
def test_inputs_that_record(dev, name):
    call, ins = calls(dev)[name]
    want = call(*ins)
    for i in range(len(ins)):
        leaf = [t.clone().requires_grad_(j == i) for j, t in enumerate(ins)]
        with pytest.raises(ValueError, match="no gradient"):
            call(*leaf)
        with torch.no_grad():
            assert torch.equal(call(*leaf), want)
        with torch.inference_mode():
            assert torch.equal(call(*leaf), want)
        assert torch.equal(call(*[t.detach() for t in leaf]), want)


@pytest.mark.parametrize("name", NAMES)
def test_inputs_with_a_tangent(dev, name):
    call, ins = calls(dev)[name]
    want = call(*ins)
    with forward_ad.dual_level():
        for i in range(len(ins)):
            dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(ins)]
            with pytest.raises(ValueError, match="no gradient"):
                call(*dual)
        assert torch.equal(call(*ins), want)
