"""Linears with 4-bit weights, for projections of a few tokens.

``FourBitLinear`` holds an ``nn.Linear`` in ``kernels.fourbit``'s int4 or mxfp4: about a quarter of the bf16 weight's
bytes, which are its time where the rows are few.  ``quantize_linears`` puts it in the place of chosen linears of
any module.  The reference has no 4-bit weights; there is no reference counterpart.
"""
import torch
from torch import nn

from qwen_image_accel.kernels import fourbit
from qwen_image_accel.kernels.adapters import takes_rows


def convertible(linear, kind="int4", group=64):
    """Whether ``linear`` becomes a FourBitLinear: a known kind and group, in_features a multiple of the group, a weight that is not
    empty."""
    group = fourbit.MX_GROUP if kind == "mxfp4" else group
    return (kind in fourbit.KINDS and group in fourbit.GROUPS and isinstance(linear, nn.Linear) and linear.in_features % group == 0
            and linear.weight.numel() > 0)


class FourBitLinear(nn.Module):
    """A linear held in 4 bits: ``kind`` "int4" (``group`` 32, 64 or 128; ``symmetric``: no zero points) or "mxfp4".

    Buffers: ``codes``, ``scales``, ``zeros`` (or None) in the kernels' layout, and ``bias`` (bf16, or None); a state dict
    holds them as they are.  They keep their types when the model around them is cast."""

    def __init__(self, linear, kind="int4", group=64, *, symmetric=False):
        super().__init__()
        weight = fourbit.quantize_weight(linear.weight.detach(), kind, group, symmetric=symmetric)
        bias = None if linear.bias is None else linear.bias.detach().to(torch.bfloat16).contiguous()
        self._hold(weight, bias)

    def _hold(self, weight, bias):
        self.in_features, self.out_features, self.group = weight.width, weight.rows, weight.group
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("zeros", weight.zeros)
        self.register_buffer("bias", bias)

    @classmethod
    def from_packed(cls, weight, bias=None):
        """A ``FourBitLinear`` over a ``kernels.fourbit.FourBitWeight`` (a checkpoint's codes: ``pack_weight``)."""
        self = cls.__new__(cls)
        nn.Module.__init__(self)
        self._hold(weight, bias)
        return self

    @property
    def packed(self):
        """The ``FourBitWeight`` of the buffers."""
        return fourbit.FourBitWeight(self.codes, self.scales, self.zeros, self.out_features, self.in_features, self.group)

    def _apply(self, fn, recurse=True):
        kept = dict(self.named_buffers(recurse=False))
        super()._apply(fn, recurse)
        for name, t in kept.items():
            moved = getattr(self, name)
            if moved.dtype != t.dtype:
                setattr(self, name, t.to(moved.device))
        return self

    def forward(self, x):
        rows = x.reshape(-1, self.in_features)
        if not takes_rows(rows):
            rows = rows.clone(memory_format=torch.contiguous_format)
        return fourbit.matmul(rows, self.packed, bias=self.bias).view(*x.shape[:-1], self.out_features)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, kind={self.packed.kind}, group={self.group}"


def quantize_linears(module, names, kind="int4", group=64, *, symmetric=False):
    """Replace the ``nn.Linear`` s of ``module`` at the given paths ("time_embed.linear_1", ...) by ``FourBitLinear`` s.
    Returns the paths, each once.  A path that is no convertible linear, or whose weight cannot be quantized, is refused before
    any is replaced."""
    names = list(dict.fromkeys(names))
    for name in names:
        if not name or not convertible(module.get_submodule(name), kind, group):
            raise ValueError(f"{name!r} is not a linear whose in_features are a multiple of its {kind} group ({group})")
    with torch.no_grad():
        made = [FourBitLinear(module.get_submodule(name), kind, group, symmetric=symmetric) for name in names]
    for name, linear in zip(names, made):
        parent, _, leaf = name.rpartition(".")
        setattr(module.get_submodule(parent), leaf, linear)
    return names


__all__ = ["FourBitLinear", "convertible", "quantize_linears"]
