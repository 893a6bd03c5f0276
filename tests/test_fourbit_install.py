"""quantize_linears refuses before it replaces anything; convertible knows kinds and groups; weights of other types (no GPU)."""
import pytest
import torch
from torch import nn

from qwen_image_accel.kernels import fourbit
from qwen_image_accel.optimizations.fourbit import FourBitLinear, convertible, quantize_linears


def net():
    torch.manual_seed(0)
    return nn.Sequential(nn.Linear(128, 8), nn.Sequential(nn.Linear(64, 8), nn.Linear(64, 8)))


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("kind", ["int4", "mxfp4"])
def test_a_later_weight_that_cannot_be_quantized_leaves_all_as_they_were(kind, bad):
    m = net()
    before = dict(m.named_modules())
    with torch.no_grad():
        m[1][1].weight[3, 5] = bad
    with pytest.raises(ValueError):
        quantize_linears(m, ["0", "1.0", "1.1"], kind)
    assert dict(m.named_modules()) == before


def test_a_path_given_twice_is_replaced_once():
    m = net()
    assert quantize_linears(m, ["0", "1.1", "0"]) == ["0", "1.1"]
    assert isinstance(m[0], FourBitLinear) and isinstance(m[1][0], nn.Linear) and isinstance(m[1][1], FourBitLinear)


@pytest.mark.parametrize("names,kw", [(["0", ""], {}), (["0", "1"], {}), (["0"], dict(kind="nf4")), (["0"], dict(group=16)), (["0"], dict(group=0)),
                                      (["0"], dict(group=-64)), (["0", "1.0"], dict(group=128))])
def test_refusals(names, kw):
    m = net()
    before = dict(m.named_modules())
    with pytest.raises(ValueError):
        quantize_linears(m, names, **kw)
    assert dict(m.named_modules()) == before


def test_the_root_is_refused():
    with pytest.raises(ValueError):
        quantize_linears(nn.Linear(64, 8), [""])


def test_convertible():
    linear = nn.Linear(256, 8)
    assert all(convertible(linear, "int4", g) for g in (32, 64, 128)) and convertible(linear, "mxfp4", 7)
    assert not any(convertible(linear, "int4", g) for g in (0, -64, 16, 256)) and not convertible(linear, "nf4", 64)
    assert not convertible(nn.Linear(64, 0)) and not convertible(nn.Linear(0, 8))


@pytest.mark.parametrize("kw", [dict(), dict(symmetric=True), dict(kind="mxfp4")])
def test_float64_weights(kw):
    w = torch.randn(16, 64, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    for a, b in zip(fourbit.quantize_weight(w, **kw)[:3], fourbit.quantize_weight(w.float(), **kw)[:3]):
        assert (a is None and b is None) or torch.equal(a, b)
    w[3, 5] = 1e39                                            # finite, beyond fp32
    with pytest.raises(ValueError):
        fourbit.quantize_weight(w, **kw)
