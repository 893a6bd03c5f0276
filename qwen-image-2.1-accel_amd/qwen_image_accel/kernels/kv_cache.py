"""A layer's K/V cache in MXFP8: quantized as it is written, read back in bf16.

The reference keeps the prefix K/V of cached decode in bf16 (the
``layer_cache`` of its blocks); there is no reference counterpart.  Here B
sequences hold C positions of H heads each as E4M3 codes with one E8M0
exponent per 32 values of a head row: 1.03 bytes a value.  The codes and
exponents are those of ``mxfp8.quantize`` on the same rows, and reading back
is exact, so the values are the same wherever the cache is read: staged by
``read_cache``, in front of a step's keys by
``attention.prepare_attention_inputs_quantized``, or in place by
``attention.attention_cached``.
"""
from typing import NamedTuple

import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels.mxfp8 import BLOCK


class QuantizedCache(NamedTuple):
    """K and V of B sequences x C positions x H heads in MXFP8, contiguous."""

    k: torch.Tensor           # (B, C, H, D) float8_e4m3fn codes
    k_exponent: torch.Tensor  # (B, C, H, D / 32) uint8, E8M0
    v: torch.Tensor
    v_exponent: torch.Tensor


def empty_cache(batch, capacity, heads, head_dim, device):
    """An uninitialised cache (its positions are to be written before they are read)."""
    if head_dim % BLOCK:
        raise ValueError(f"head dim {head_dim} is not a multiple of {BLOCK}")
    shape = (batch, capacity, heads, head_dim)
    blocks = shape[:3] + (head_dim // BLOCK,)
    return QuantizedCache(torch.empty(shape, dtype=torch.float8_e4m3fn, device=device),
                          torch.empty(blocks, dtype=torch.uint8, device=device),
                          torch.empty(shape, dtype=torch.float8_e4m3fn, device=device),
                          torch.empty(blocks, dtype=torch.uint8, device=device))


def check_cache(name, cache):
    """(B, C, H, D) of a cache the kernels can read, else Unsupported."""
    k, ke, v, ve = cache
    shape, device = k.shape, k.device
    if k.dim() != 4 or shape[3] % BLOCK or not k.is_cuda:
        raise _native.Unsupported(name, _native.QIM_ERR_LAYOUT, "the cache holds (B, C, H, D) codes on the GPU")
    blocks = shape[:3] + (shape[3] // BLOCK,)
    if not (k.dtype == v.dtype == torch.float8_e4m3fn and ke.dtype == ve.dtype == torch.uint8 and v.shape == shape
            and ke.shape == blocks and ve.shape == blocks and ke.device == v.device == ve.device == device
            and k.is_contiguous() and ke.is_contiguous() and v.is_contiguous() and ve.is_contiguous()):
        raise _native.Unsupported(name, _native.QIM_ERR_LAYOUT,
                                  "codes (B, C, H, D) float8_e4m3fn and exponents (B, C, H, D/32) uint8, contiguous, "
                                  "on one device")
    return shape


def per_sequence(name, what, t, batch, device):
    """The address of a (B,) int32 device tensor."""
    if (not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.shape != (batch,) or t.device != device
            or not t.is_contiguous()):
        raise _native.Unsupported(name, _native.QIM_ERR_LAYOUT, f"{what} is a contiguous int32 ({batch},) tensor on {device}")
    return t.data_ptr()


def token_strides(t):
    """(elements between sequences, elements between tokens) of a (B, S, H, D)
    tensor with packed heads, else None.  The stride of an axis of one element
    says nothing and is not looked at."""
    b, s, h, d = t.shape
    batch, token, head, one = t.stride()
    if (d > 1 and one != 1) or (h > 1 and head != d):
        return None
    if s == 1:
        token = h * d
    return (batch if b > 1 else s * token), token


def write_cache(cache, k, v, start=0, count=None):
    """Quantize K and V rows (B, S, H, D) bf16 into ``cache``: row s of sequence
    b to position start[b] + s.

    ``start``: an int for every sequence (the rows have to fit), or an int32
    (B,) device tensor, as a captured step needs it.  ``count``: None, or
    an int32 (B,) device tensor: only the first count[b] rows are written (a
    padded batch).  With device tensors, rows whose position is outside the
    cache are not written.  Positions not written keep their values.  k, v: packed heads,
    any token and batch stride (e.g. views into a fused QKV output)."""
    b, c, h, d = check_cache("write_cache", cache)
    device = cache.k.device
    shape = k.shape
    s = shape[1] if len(shape) == 4 else 0
    strides = ()
    for t in (k, v):
        step = token_strides(t) if t.dtype == torch.bfloat16 and t.device == device and t.shape == (b, s, h, d) else None
        if step is None:
            raise _native.Unsupported("write_cache", _native.QIM_ERR_LAYOUT,
                                      f"k and v are bf16 ({b}, S, {h}, {d}) tensors with packed heads on {device}")
        strides += step
    if not (b and s and h and d):
        return
    counts = None if count is None else per_sequence("write_cache", "count", count, b, device)
    if isinstance(start, torch.Tensor):
        starts, first = per_sequence("write_cache", "start", start, b, device), 0
        if c == 0:
            return
    else:
        starts, first = None, int(start)
        if not 0 <= first <= c - s:
            raise _native.QimError("write_cache", _native.QIM_ERR_ARG, f"{s} rows from position {first} of {c}")
    _native.call_on(device, "qim_cache_write", k.data_ptr(), *strides[:2], v.data_ptr(), *strides[2:],
                    cache.k.data_ptr(), cache.k_exponent.data_ptr(), cache.v.data_ptr(), cache.v_exponent.data_ptr(), starts, first, counts, b, s, c, h, d)


def read_cache(cache, rows=None):
    """(K, V), each (B, rows, H, D) bf16: the values of the first ``rows``
    positions (default: all) of every sequence."""
    b, c, h, d = check_cache("read_cache", cache)
    rows = c if rows is None else int(rows)
    if not 0 <= rows <= c:
        raise ValueError(f"{rows} rows of a cache of {c} positions")
    device = cache.k.device
    k = torch.empty((b, rows, h, d), dtype=torch.bfloat16, device=device)
    v = torch.empty_like(k)
    if rows and k.numel():
        _native.call_on(device, "qim_cache_read", cache.k.data_ptr(), cache.k_exponent.data_ptr(), cache.v.data_ptr(),
                        cache.v_exponent.data_ptr(), k.data_ptr(), v.data_ptr(), b, c, rows, h, d)
    return k, v
