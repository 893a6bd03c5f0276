"""The prefix K/V of cached decode held in MXFP8.

The reference's blocks keep each layer's prefix K/V (text and condition
tokens, computed once) in a bf16 ``layer_cache`` and put it in front of every
step's keys.  ``quantize_layer_cache`` holds it in MXFP8 instead (1.03 bytes a
value for 2): pass its result as ``layer_cache``, and the cached-decode
processors read it in the fused norm + RoPE + pack kernel.  There is no
reference counterpart.
"""
import torch

from qwen_image_accel.kernels.kv_cache import empty_cache, read_cache, token_strides, write_cache


def _writable(t):
    """t, or a copy where ``write_cache`` does not take its rows as they lie."""
    strides = token_strides(t)
    ok = strides is not None and strides[1] >= t.shape[2] * t.shape[3] and not (strides[0] % 8 or strides[1] % 8 or t.data_ptr() % 16)
    return t if ok else t.clone(memory_format=torch.contiguous_format)


class QuantizedLayerCache:
    """A ``layer_cache`` over (B, P, H, D) bf16 K and V, kept in MXFP8
    (``quantized``, a ``kernels.kv_cache.QuantizedCache``)."""

    def __init__(self, k, v):
        if k.shape != v.shape or k.dim() != 4:
            raise ValueError(f"prefix K and V must both be (B, P, H, D), got {tuple(k.shape)} and {tuple(v.shape)}")
        b, p, h, d = k.shape
        self.quantized = empty_cache(b, p, h, d, k.device)
        write_cache(self.quantized, _writable(k), _writable(v))

    def get(self):
        """The prefix in bf16, for a consumer that takes no MXFP8."""
        return read_cache(self.quantized)


def quantize_layer_cache(layer_cache):
    """``layer_cache`` (anything whose ``get()`` returns the prefix K and V) as
    a ``QuantizedLayerCache``; itself if it is one."""
    if isinstance(layer_cache, QuantizedLayerCache):
        return layer_cache
    return QuantizedLayerCache(*layer_cache.get())


__all__ = ["QuantizedLayerCache", "quantize_layer_cache"]
