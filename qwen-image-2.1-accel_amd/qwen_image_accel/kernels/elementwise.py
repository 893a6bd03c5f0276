"""BF16 gated residual and complex rotary embedding.

Reference interface: src/qwen_image_accel/kernels/elementwise.py --
``residual(h, x, gate)`` (:26-34) and ``rope_qk(q, k, freqs)`` (:63-69).
Kernels: libqim's ``qim_gated_residual`` and ``qim_rope_qk``.
``residual_norm`` (no reference counterpart) is the residual with the norms on
both sides of it in one pass: libqim's ``qim_residual_norm``.
"""
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels.adapters import row_layout
from qwen_image_accel.kernels.bf16 import HEAD_DIMS
from qwen_image_accel.kernels.mxfp8 import empty_quantized


def residual(h, x, gate):
    """``h + gate * x`` with the product rounded to bf16 before the add.

    h, x: (B, S, D); gate: (B, 1, D).  Unsupported inputs take the eager path
    (reference guard, kernels/elementwise.py:27-28)."""
    if (h.dtype == torch.bfloat16 and h.is_contiguous() and x.is_contiguous() and h.is_cuda
            and h.ndim == 3 and x.shape == h.shape and x.dtype == torch.bfloat16
            and x.device == h.device and gate.dtype == torch.bfloat16 and gate.device == h.device
            and gate.shape == (h.shape[0], 1, h.shape[2]) and gate.is_contiguous()
            and h.shape[-1] % 8 == 0 and h.numel() > 0):
        b, s, d = h.shape
        out = torch.empty_like(h)
        _native.call("qim_gated_residual", _native.ptr(h), _native.ptr(x), _native.ptr(gate),
                     _native.ptr(out), b * s, d, s, _native.stream(h.device))
        return out
    return h + gate * x


def norm_kind(norm):
    """``NORM_LAYER``, ``NORM_RMS`` or ``NORM_NONE`` (None) of what ``residual_norm`` takes as a norm, else None.

    A module counts by its class, since others with the same attributes compute other things: torch's LayerNorm, or one that is
    named after it, and torch's RMSNorm with its own ``forward``, or a class named RMSNorm (Diffusers', x / rms times the weight).
    Any other object holds a norm's parameters: with a ``normalized_shape`` a LayerNorm's, else an RMSNorm's."""
    if norm is None:
        return _native.NORM_NONE
    shaped = getattr(norm, "normalized_shape", None) is not None
    if not isinstance(norm, torch.nn.Module):
        return _native.NORM_LAYER if shaped else _native.NORM_RMS
    cls = type(norm)
    if isinstance(norm, torch.nn.RMSNorm):
        return _native.NORM_RMS if cls.forward is torch.nn.RMSNorm.forward else None
    if isinstance(norm, torch.nn.LayerNorm) or (shaped and cls.__name__.endswith("LayerNorm")):
        return _native.NORM_LAYER
    return _native.NORM_RMS if cls.__name__ == "RMSNorm" and not shaped else None


def _norm_of(norm, d, device, refuse):
    """(kind, weight or None, eps) of a norm over d values that ``residual_norm`` takes."""
    kind = norm_kind(norm)
    if kind == _native.NORM_NONE:
        return kind, None, 0.0
    if kind is None:
        refuse(f"a {type(norm).__name__} is no LayerNorm or RMSNorm")
    weight, eps = getattr(norm, "weight", None), getattr(norm, "eps", None)
    if eps is None or getattr(norm, "bias", None) is not None:
        refuse("a norm has an eps and no bias")
    shape = getattr(norm, "normalized_shape", None)
    if shape is not None and tuple(shape) != (d,):
        refuse(f"a norm over {tuple(shape)} of rows of {d}")
    if kind == _native.NORM_LAYER:
        if weight is not None or getattr(norm, "elementwise_affine", False):
            refuse("a LayerNorm has no affine")
        return kind, None, float(eps)
    if weight is not None and (weight.shape != (d,) or weight.dtype != torch.bfloat16 or weight.device != device
                               or not weight.is_contiguous()):
        refuse(f"an RMSNorm's weight is a contiguous bf16 ({d},) tensor on {device}")
    return kind, weight, float(eps)


def residual_norm(h, x, norm, *, gate=None, residual_scale=1.0, post=None, scale=None, shift=None, add_one=False,
                  quantized=False, tiled=False, rounding="once", out=None):
    """The end of one block branch and the start of the next in one pass:

        h' = h + residual_scale * gate * post(x),   z = norm(h') * scale + shift

    Returns (h', z).  h, x: (B, S, D) or (M, D) bf16 on the GPU, fewer than 2^22 rows any multiple of 8 elements apart, D
    a multiple of 8 up to 16384.  ``norm`` and ``post`` (None: x itself): an RMSNorm (``weight`` bf16 or
    None, ``eps``) or a LayerNorm without affine (``normalized_shape``, ``eps``); ``norm_kind`` says what counts as which, other
    modules are refused.  ``gate``, ``scale``, ``shift``: None, (B, 1, D) bf16, one vector per sequence at any stride that is
    a multiple of 8, or one for all, (1, 1, D) or (D,).
    ``add_one``: 1 + scale instead of scale.  z is a new bf16 tensor, or with ``quantized`` a
    ``mxfp8.Quantized`` (``tiled``: in the GEMM's layout; D a multiple of 128).  ``out``: where h' goes, by default a
    new tensor; h or x itself is fine, else it shares no rows with them, and nothing with the vectors and weights.

    ``rounding="once"``: fp32 throughout, h' and z rounded at their ends (z from the unrounded h').
    ``"eager"``: the bits of ``residual(h, x, gate)`` followed by ``layernorm.layer_norm_scale`` or
    ``epilogue.layer_norm_scale_quantize`` on its result; for a gate and a scale, a LayerNorm, no post and a
    residual_scale of 1.  No gradient is recorded."""
    def refuse(why):
        raise _native.Unsupported("residual_norm", _native.QIM_ERR_LAYOUT, why)
    device, shape = h.device, h.shape
    if not h.is_cuda:
        refuse("expects tensors on the GPU")
    if rounding not in ("once", "eager"):
        raise ValueError(f"rounding={rounding!r}: once or eager")
    if norm is None:
        raise ValueError("residual_norm needs the norm that follows the residual")

    def rows(t):
        lay = row_layout(t) if t.dtype == torch.bfloat16 and t.shape == shape and t.device == device else None
        if lay is None:
            refuse(f"h, x and out are bf16 {tuple(shape)} tensors on {device} with rows one stride apart")
        return lay
    if len(shape) not in (2, 3):
        refuse("h is a (B, S, D) or (M, D) tensor")
    m, d, ldh = rows(h)
    ldx = rows(x)[2]
    batch = shape[0] if len(shape) == 3 else 1

    def vector(t):
        """(address, elements between sequences)"""
        if t is None:
            return None, 0
        if t.dtype != torch.bfloat16 or t.device != device or t.shape not in ((batch, 1, d), (1, 1, d), (d,)) or (d > 1 and t.stride(-1) != 1):
            refuse(f"gate, scale and shift are bf16 ({batch}, 1, {d}), (1, 1, {d}) or ({d},) tensors on {device}")
        return t.data_ptr(), t.stride(0) if t.dim() == 3 and t.shape[0] > 1 else 0
    post_kind, post_w, post_eps = _norm_of(post, d, device, refuse)
    norm_kind, norm_w, norm_eps = _norm_of(norm, d, device, refuse)
    vectors = vector(gate) + vector(scale) + vector(shift)
    if out is None:
        out, ldo = torch.empty_like(h, memory_format=torch.contiguous_format), d
    else:
        ldo = rows(out)[2]
    if quantized:
        z = empty_quantized(m, d, device, shape, tiled)
        z_ptr, z_scales = z.values.data_ptr(), z.scales.data_ptr()
    else:
        z = torch.empty_like(h, memory_format=torch.contiguous_format)
        z_ptr, z_scales = z.data_ptr(), None
    if m == 0 or d == 0:
        return out, z
    flags = ((_native.ADALN_ADD_ONE if add_one and scale is not None else 0) | (_native.ADALN_TILED if quantized and tiled else 0)
             | (_native.NORM_EAGER if rounding == "eager" else 0))
    _native.call_on(device, "qim_residual_norm", h.data_ptr(), ldh, x.data_ptr(), ldx, post_kind, _native.ptr(post_w), post_eps,
                    *vectors[:2], float(residual_scale), norm_kind, _native.ptr(norm_w), norm_eps, *vectors[2:], flags,
                    out.data_ptr(), ldo, z_ptr, d, z_scales, m, d, shape[1] if len(shape) == 3 else m)
    return out, z


MOD_COPY, MOD_ONE_PLUS, MOD_TANH = 0, 1, 2


def modulation_values(mod, kinds):
    """The per-step modulation terms (reference optimizations/fusion.py:48-53,
    ``1 + s`` and ``tanh(g)`` of the modulation chunks) in one launch.

    mod: (..., P, D) contiguous bf16 on the GPU; row i of each group of P rows
    is copied (MOD_COPY), mapped to bf16(1 + x) (MOD_ONE_PLUS) or to
    bf16(tanh(x)) (MOD_TANH; tanh in float64, rounded to fp32, then to bf16),
    i.e. kinds[i].  Returns (P, ..., D): term i is the contiguous ``out[i]``."""
    p, d = len(kinds), mod.shape[-1]
    if not (mod.is_cuda and mod.dtype == torch.bfloat16 and mod.is_contiguous() and mod.ndim >= 2
            and mod.shape[-2] == p and 1 <= p <= 16 and d % 8 == 0 and mod.numel() > 0
            and all(k in (MOD_COPY, MOD_ONE_PLUS, MOD_TANH) for k in kinds)):
        raise _native.Unsupported("modulation_values", _native.QIM_ERR_ARG,
                                  f"{tuple(mod.shape)} {mod.dtype} kinds={kinds}")
    out = torch.empty((p,) + tuple(mod.shape[:-2]) + (d,), dtype=mod.dtype, device=mod.device)
    bits = sum(k << (2 * i) for i, k in enumerate(kinds))
    _native.call("qim_modulation_values", _native.ptr(mod), mod.numel() // d, d, bits, p, _native.ptr(out),
                 _native.stream(mod.device))
    return out


def rope_qk(q, k, freqs):
    """Complex RoPE of q and k (B, S, H, D) with freqs (S, D/2) complex64.

    Unguarded like the reference: expects contiguous CUDA bf16 q, k."""
    out_q, out_k = torch.empty_like(q), torch.empty_like(k)
    b, s, h, d = q.shape
    if d not in HEAD_DIMS:
        raise _native.Unsupported("rope_qk", _native.QIM_ERR_SHAPE, f"head dim {d}")
    f = freqs.contiguous()
    _native.call("qim_rope_qk", _native.ptr(q), _native.ptr(k), _native.complex_ptr(f),
                 _native.ptr(out_q), _native.ptr(out_k), b, s, h, d, _native.stream(q.device))
    return out_q, out_k
