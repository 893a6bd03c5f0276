"""FourBitLinear: what it holds, how it is saved, cast and installed (no GPU needed), and its products (GPU)."""
import pytest
import torch
from torch import nn

from qwen_image_accel import _native
from qwen_image_accel.kernels import fourbit
from qwen_image_accel.optimizations.fourbit import FourBitLinear, convertible, quantize_linears
from tests import few_tokens_ref as R


def linear(k=256, n=48, bias=True, seed=0):
    torch.manual_seed(seed)
    return nn.Linear(k, n, bias=bias, dtype=torch.bfloat16)


@pytest.mark.parametrize("kind,group,symmetric", [("int4", 64, False), ("int4", 128, True), ("mxfp4", 32, False)])
def test_holds_the_quantized_weight(kind, group, symmetric):
    base = linear()
    m = FourBitLinear(base, kind, group, symmetric=symmetric)
    want = fourbit.quantize_weight(base.weight, kind, group, symmetric=symmetric)
    assert (m.in_features, m.out_features, m.group) == (256, 48, group) and m.packed.kind == kind
    for a, b in zip(m.packed[:3], want[:3]):
        assert (a is None and b is None) or torch.equal(a, b)
    assert torch.equal(m.bias, base.bias) and not list(m.parameters())
    assert FourBitLinear(linear(bias=False)).bias is None


def test_state_dicts_and_casts():
    m, other = FourBitLinear(linear(seed=1)), FourBitLinear(linear(seed=2))
    other.load_state_dict(m.state_dict())
    for a, b in zip(m.packed[:3], other.packed[:3]):
        assert torch.equal(a, b)
    types = [t.dtype for t in m.buffers()]
    for cast in (lambda x: x.float(), lambda x: x.half(), lambda x: x.to(torch.float64)):
        cast(nn.Sequential(m))
        assert [t.dtype for t in m.buffers()] == types
    assert torch.equal(m.scales, other.scales)
    again = FourBitLinear.from_packed(m.packed, m.bias)
    assert again.packed == m.packed or all(torch.equal(a, b) for a, b in zip(again.packed[:3], m.packed[:3]))


def test_quantize_linears():
    class Net(nn.Module):
        def __init__(self):
            super().__init__()
            self.a, self.b = linear(), nn.Sequential(linear(128, 8), nn.Linear(40, 8))
    net = Net()
    with pytest.raises(ValueError, match="b.1"):
        quantize_linears(net, ["a", "b.1"])
    assert isinstance(net.a, nn.Linear)                       # nothing was replaced
    assert quantize_linears(net, ["a", "b.0"], "mxfp4") == ["a", "b.0"]
    assert isinstance(net.a, FourBitLinear) and isinstance(net.b[0], FourBitLinear) and isinstance(net.b[1], nn.Linear)
    assert convertible(linear()) and not convertible(nn.Linear(96, 8)) and convertible(nn.Linear(96, 8), "mxfp4") and not convertible(nn.ReLU())


def test_host_tensors_are_refused():
    with pytest.raises(_native.Unsupported):
        FourBitLinear(linear())(torch.zeros(2, 256, dtype=torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(256,), (3, 256), (2, 5, 256), (2, 3, 7, 256), (0, 256)])
def test_products(dev, shape):
    print("[case] linear", shape, flush=True)
    m = FourBitLinear(linear()).to(dev)
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    got = m(x)
    assert got.shape == shape[:-1] + (48,) and got.dtype == torch.bfloat16
    y, e = R.four_bit(x.reshape(-1, 256), *fourbit.unpack_weight(m.packed), bias=m.bias)
    assert ((got.reshape(-1, 48).double().cpu() - y).abs() <= R.rounded(y, e)).all()


@pytest.mark.gpu
def test_rows_that_the_kernel_does_not_take_as_they_lie(dev):
    print("[case] linear strides", flush=True)
    m = FourBitLinear(linear()).to(dev)
    base = torch.randn(6, 2 * 256 + 3, device=dev).to(torch.bfloat16)
    for x in (base[:, 1:257], base[:, :512:2], base[:, :256].t().contiguous().t()):
        assert torch.equal(m(x), m(x.contiguous()))
