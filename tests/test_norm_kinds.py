"""Which norms residual_norm takes for which formula (no GPU), and that it refuses the others (GPU)."""
import types

import pytest
import torch
from torch import nn

from qwen_image_accel import _native
from qwen_image_accel.block import _LayerNorm
from qwen_image_accel.kernels import elementwise
from tests import fake_qwen21 as fq
from tests.helpers import bf16_randn

NONE, RMS, LAYER = _native.NORM_NONE, _native.NORM_RMS, _native.NORM_LAYER


class UnitOffset(nn.RMSNorm):
    """x / rms * (1 + weight)."""

    def forward(self, x):
        return nn.functional.rms_norm(x, self.normalized_shape, None, self.eps) * (1 + self.weight)


class OffsetRMSNorm(nn.Module):
    """The same as a module of its own, with an RMSNorm's attributes."""

    def __init__(self, dim, eps=1e-6):
        super().__init__()
        self.weight, self.eps = nn.Parameter(torch.zeros(dim)), eps


class ShapedRMSNorm(nn.Module):
    """An RMSNorm with a LayerNorm's attributes."""

    def __init__(self, dim):
        super().__init__()
        self.normalized_shape, self.elementwise_affine, self.eps = (dim,), False, 1e-6


class CastLayerNorm(nn.LayerNorm):
    def forward(self, x):
        return super().forward(x.float()).to(x.dtype)


WRONG = [nn.GroupNorm(1, 64, affine=False), nn.InstanceNorm1d(64), nn.BatchNorm1d(64, affine=False), UnitOffset(64, eps=1e-6), OffsetRMSNorm(64),
         ShapedRMSNorm(64)]


@pytest.mark.parametrize("norm,kind", [
    (None, NONE), (nn.LayerNorm(64, elementwise_affine=False), LAYER), (CastLayerNorm(64, elementwise_affine=False), LAYER),
    (_LayerNorm(64), LAYER), (nn.RMSNorm(64, eps=1e-6), RMS), (nn.RMSNorm(64, eps=1e-6, elementwise_affine=False), RMS), (fq.RMSNorm(64), RMS),
    (types.SimpleNamespace(weight=None, eps=1e-6), RMS), (types.SimpleNamespace(normalized_shape=(64,), eps=1e-6), LAYER)]
    + [(n, None) for n in WRONG], ids=lambda v: type(v).__name__ if isinstance(v, nn.Module) else str(v)[:20])
def test_kinds(norm, kind):
    assert elementwise.norm_kind(norm) == kind


@pytest.mark.gpu
@pytest.mark.parametrize("norm", WRONG, ids=lambda v: type(v).__name__)
def test_other_norms_are_refused(dev, norm):
    print("[case] norm", type(norm).__name__, flush=True)
    norm = norm.to(dev).to(torch.bfloat16)
    h, x = (bf16_randn(torch.Generator().manual_seed(i), (2, 3, 64)).to(dev) for i in range(2))
    with pytest.raises(_native.Unsupported):
        elementwise.residual_norm(h, x, norm)
    with pytest.raises(_native.Unsupported):
        elementwise.residual_norm(h, x, nn.LayerNorm(64, elementwise_affine=False), post=norm)


@pytest.mark.gpu
def test_a_module_of_a_known_class(dev):
    """The same bits from a module as from its parameters."""
    print("[case] norm modules", flush=True)
    h, x = (bf16_randn(torch.Generator().manual_seed(i), (2, 3, 64)).to(dev) for i in range(2))
    w = bf16_randn(torch.Generator().manual_seed(2), (64,)).to(dev)
    want = elementwise.residual_norm(h, x, types.SimpleNamespace(weight=w, eps=1e-6))
    for norm in (nn.RMSNorm(64, eps=1e-6), fq.RMSNorm(64)):
        norm = norm.to(dev).to(torch.bfloat16)
        norm.weight.data.copy_(w)
        got = elementwise.residual_norm(h, x, norm)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
