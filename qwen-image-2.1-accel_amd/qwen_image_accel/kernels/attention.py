"""Fused Q/K RMSNorm + RoPE + prefix K/V packing of cached decode.

Reference interface: src/qwen_image_accel/kernels/attention.py:92-159
``prepare_attention_inputs(q, k, v, norm_q, norm_k, freqs, cached_k, cached_v)``
-> ``(rope(norm_q(q)), cat[ck, rope(norm_k(k))], cat[cv, v])`` or ``None``.
Kernel: libqim's ``qim_qk_norm_rope_pack``; any head count (the reference's
kernel is fixed to 32 x 128) and head dims 64/128/256.  No buffer persists
across calls.
"""
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import kv_cache, mxfp8
from qwen_image_accel.kernels.bf16 import HEAD_DIMS


def _norm_ok(norm, d, device):
    w = getattr(norm, "weight", None)
    return (w is not None and getattr(norm, "bias", None) is None and w.shape == (d,)
            and w.dtype == torch.bfloat16 and w.device == device and w.is_contiguous())


def _prepare_layout(q, k, v, norm_q, norm_k, freqs):
    """(b, s, h, d, token stride) of the step's own operands, or None where the
    kernel does not take them."""
    if (q.ndim != 4 or q.shape[-1] not in HEAD_DIMS or q.shape[1] == 0
            or k.shape != q.shape or v.shape != q.shape
            or freqs is None or freqs.dtype != torch.complex64
            or freqs.shape != (q.shape[1], q.shape[-1] // 2) or not freqs.is_contiguous()
            or freqs.device != q.device):
        return None
    # q, k, v: contiguous, or column blocks of one fused QKV output -- packed
    # heads and one token stride shared by the three (the kernel's ldt).
    b, s, h, d = q.shape
    ldt = q.stride(1)
    for t in (q, k, v):
        if t.dtype != torch.bfloat16 or not t.is_cuda or t.device != q.device or t.stride() != (s * ldt, ldt, d, 1):
            return None
    if not (_norm_ok(norm_q, d, q.device) and _norm_ok(norm_k, d, q.device)):
        return None
    return b, s, h, d, ldt


def _prepare_outputs(q, prefix):
    b, s, h, d = q.shape
    oq = torch.empty((b, s, h, d), device=q.device, dtype=q.dtype)
    ok = torch.empty((b, s + prefix, h, d), device=q.device, dtype=q.dtype)
    return oq, ok, torch.empty_like(ok)


def prepare_attention_inputs(q, k, v, norm_q, norm_k, freqs, cached_k, cached_v):
    """Return fused Q/K/V, or None when the original operators should be used."""
    if (q.ndim != 4 or cached_k.ndim != 4 or cached_k.shape[0] != q.shape[0]
            or cached_k.shape[2:] != q.shape[2:] or cached_v.shape != cached_k.shape):
        return None
    for t in (cached_k, cached_v):
        if t.dtype != torch.bfloat16 or not t.is_cuda or t.device != q.device or not t.is_contiguous():
            return None
    layout = _prepare_layout(q, k, v, norm_q, norm_k, freqs)
    if layout is None:
        return None
    b, s, h, d, ldt = layout
    p = cached_k.shape[1]
    oq, ok, ov = _prepare_outputs(q, p)
    _native.call("qim_qk_norm_rope_pack", _native.ptr(q), _native.ptr(k), _native.ptr(v),
                 _native.ptr(cached_k) if p else None, _native.ptr(cached_v) if p else None,
                 _native.ptr(norm_q.weight), _native.ptr(norm_k.weight), _native.complex_ptr(freqs),
                 _native.ptr(oq), _native.ptr(ok), _native.ptr(ov), b, s, p, h, d, ldt,
                 float(norm_q.eps), float(norm_k.eps), _native.stream(q.device))
    return oq, ok, ov


def prepare_attention_inputs_quantized(q, k, v, norm_q, norm_k, freqs, cache, prefix=None):
    """``prepare_attention_inputs`` with the prefix in an MXFP8 cache
    (``kv_cache.QuantizedCache``, of which the first ``prefix`` positions, by
    default all, are the prefix): its values go in front of k and v as
    ``kv_cache.read_cache`` gives them, without that copy.  The rotated q and k
    are rounded to bf16 once, at their end; ``prepare_attention_inputs`` rounds
    after the normalisation and after its weight too, as the reference's
    operators do.  None where the kernel does not take the step's own operands."""
    b, c, h, d = kv_cache.check_cache("prepare_attention_inputs_quantized", cache)
    p = c if prefix is None else int(prefix)
    if not 0 <= p <= c:
        raise ValueError(f"a prefix of {p} in a cache of {c} positions")
    layout = _prepare_layout(q, k, v, norm_q, norm_k, freqs)
    if layout is None or cache.k.device != q.device or (b, h, d) != (layout[0], layout[2], layout[3]):
        return None
    s, ldt = layout[1], layout[4]
    oq, ok, ov = _prepare_outputs(q, p)
    _native.call_on(q.device, "qim_qk_norm_rope_pack_cached", q.data_ptr(), k.data_ptr(), v.data_ptr(),
                    cache.k.data_ptr(), cache.k_exponent.data_ptr(), cache.v.data_ptr(), cache.v_exponent.data_ptr(), c,
                    norm_q.weight.data_ptr(), norm_k.weight.data_ptr(), _native.complex_ptr(freqs), oq.data_ptr(),
                    ok.data_ptr(), ov.data_ptr(), b, s, p, h, d, ldt, float(norm_q.eps), float(norm_k.eps))
    return oq, ok, ov


def attention_cached(q, cache, lengths, *, tree=None, scale=None, out=None):
    """softmax(q K^T * scale) V of a few tokens over an MXFP8 cache, read in
    place: libqim's ``qim_attention_cached``.

    q: (B, S, H, 128) bf16, S <= 64, packed heads, any token and batch
    stride; ``cache``: B sequences of C positions with HK heads, H a
    multiple of HK (query head h reads K/V head h // (H // HK)).  ``lengths``:
    int32 (B,) device tensor, the keys of each sequence, its own S tokens
    among them when they attend to themselves (write them with
    ``kv_cache.write_cache`` first); values outside [0, C] count as the nearest
    of the two.  ``tree``: None (every key is seen), or bool (B, S, S) or
    (S, S): of the last S keys, query i sees key j only where tree[..., i, j]
    (drafted tokens: itself and its ancestors; a causal step: the lower
    triangle).  A row that sees no key is zeros (all are, of a cache of no positions).  scale defaults to
    1/sqrt(128).  Returns (B, S, H, 128) bf16 (``out``, if given: contiguous, apart from q).  For the queries of a whole image,
    stage the prefix (``prepare_attention_inputs_quantized``) and use
    ``attention``."""
    b, c, kv, d = kv_cache.check_cache("attention_cached", cache)
    device = cache.k.device
    shape = q.shape
    strides = (kv_cache.token_strides(q) if len(shape) == 4 and q.dtype == torch.bfloat16 and q.device == device
               and shape[0] == b and shape[3] == d else None)
    if strides is None:
        raise _native.Unsupported("attention_cached", _native.QIM_ERR_LAYOUT,
                                  f"q is a bf16 ({b}, S, H, {d}) tensor with packed heads on {device}")
    s, h = shape[1], shape[2]
    size = kv_cache.per_sequence("attention_cached", "lengths", lengths, b, device)
    mask, mask_b = None, 0
    if tree is not None:
        if tree.dtype != torch.bool or tree.device != device or tree.shape not in ((s, s), (b, s, s)) or not tree.is_contiguous():
            raise _native.Unsupported("attention_cached", _native.QIM_ERR_LAYOUT,
                                      f"tree is a contiguous bool ({b}, {s}, {s}) or ({s}, {s}) tensor on {device}")
        mask, mask_b = tree.data_ptr(), s * s if tree.dim() == 3 else 0
    if out is None:
        out = torch.empty((b, s, h, d), dtype=torch.bfloat16, device=device)
    elif out.dtype != torch.bfloat16 or out.shape != shape or out.device != device or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous bf16 {tuple(q.shape)} tensor on {device}")
    if not (b and s and h and d):
        return out
    if c == 0:
        if d != 128 or s > 64 or kv == 0 or h % kv:
            raise _native.Unsupported("attention_cached", _native.QIM_ERR_SHAPE, f"{s} tokens, {h} heads of {d} on {kv} K/V heads")
        return out.zero_()
    nbytes = _native.bytes_on(device, "qim_attention_cached_workspace_bytes", b, s, c, h, kv)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _native.call_on(device, "qim_attention_cached", q.data_ptr(), *strides, cache.k.data_ptr(),
                    cache.k_exponent.data_ptr(), cache.v.data_ptr(), cache.v_exponent.data_ptr(), size, mask, mask_b,
                    out.data_ptr(), _native.ptr(ws), nbytes, b, s, c, h, kv, d,
                    float(scale if scale is not None else d ** -0.5))
    return out


def attention_shared(q, prefix, cache, lengths, *, share=None, prefix_lengths=None, tree=None, scale=None, out=None):
    """``attention_cached`` of requests that continue shared prefixes, each prefix read once for all of its
    requests: softmax(q [Kp; K]^T * scale) [Vp; V], libqim's ``qim_attention_shared``.

    q: (B, S, H, 128) bf16, S <= 64, packed heads, any token and batch stride.  ``prefix``: P prefixes of CP positions
    (CP > 0), ``cache``: the B requests' own keys, both ``kv_cache.QuantizedCache`` with HK heads.  ``share``: int32
    (B,) device tensor, the prefix of each request (any other number, -1 by convention: none), or None where P
    is 1 and every request continues it.  ``prefix_lengths``: int32 (P,) device tensor, the keys of each prefix, or None
    (all CP); ``lengths``: int32 (B,) device tensor, the own keys of each request, its S tokens among them
    when they attend to themselves.  Lengths outside the caches count as the nearest inside.
    ``tree``, ``scale`` and ``out`` as for ``attention_cached``; the tree's keys are the last S own ones.  A row that
    sees no key is zeros.  Returns (B, S, H, 128) bf16."""
    name = "attention_shared"

    def refuse(why):
        raise _native.Unsupported(name, _native.QIM_ERR_LAYOUT, why)
    p, cp, kv, d = kv_cache.check_cache(name, prefix)
    b, c, own_kv, own_d = kv_cache.check_cache(name, cache)
    device = cache.k.device
    if (own_kv, own_d) != (kv, d) or prefix.k.device != device:
        refuse(f"prefix and own cache have one number of heads and head dim, on {device}")
    if not (p and cp and kv):
        refuse("a prefix of no positions: use attention_cached")
    shape = q.shape
    strides = (kv_cache.token_strides(q) if len(shape) == 4 and q.dtype == torch.bfloat16 and q.device == device
               and shape[0] == b and shape[3] == d else None)
    if strides is None:
        refuse(f"q is a bf16 ({b}, S, H, {d}) tensor with packed heads on {device}")
    s, h = shape[1], shape[2]
    size = kv_cache.per_sequence(name, "lengths", lengths, b, device)
    psize = None if prefix_lengths is None else kv_cache.per_sequence(name, "prefix_lengths", prefix_lengths, p, device)
    if share is None and p != 1:
        refuse(f"share names the prefix of each request where there are {p}")
    which = None if share is None else kv_cache.per_sequence(name, "share", share, b, device)
    mask, mask_b = None, 0
    if tree is not None:
        if tree.dtype != torch.bool or tree.device != device or tree.shape not in ((s, s), (b, s, s)) or not tree.is_contiguous():
            refuse(f"tree is a contiguous bool ({b}, {s}, {s}) or ({s}, {s}) tensor on {device}")
        mask, mask_b = tree.data_ptr(), s * s if tree.dim() == 3 else 0
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.dtype != torch.bfloat16 or out.shape != shape or out.device != device or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous bf16 {tuple(shape)} tensor on {device}")
    if not (b and s and h):
        return out
    own = [(t if c else u).data_ptr() for t, u in zip(cache, prefix)]   # an empty cache has no address; it is not read
    nbytes = _native.bytes_on(device, "qim_attention_shared_workspace_bytes", b, s, cp, c, h, kv, p, int(share is not None))
    ws = q.new_empty(max(nbytes, 16), dtype=torch.uint8)
    _native.call_on(device, "qim_attention_shared", q.data_ptr(), *strides, *(t.data_ptr() for t in prefix), psize, which,
                    *own, size, mask, mask_b, out.data_ptr(), ws.data_ptr(), nbytes, b, s, p, cp, c, h, kv, d,
                    float(scale if scale is not None else d ** -0.5))
    return out


def workspace(b, s, t, h, device, d=128):
    """A workspace for ``attention`` / ``attention_mxfp8`` of this shape (room
    for V^T tiles first, then the split items' partial results)."""
    device = torch.get_default_device() if device is None else torch.device(device)
    if device.type != "cuda":
        raise ValueError(f"Expected a cuda device, but got: {device}")
    if device.index is None or device.index == torch.cuda.current_device():
        nbytes = _native.lib().qim_attention_workspace_bytes(b, s, t, h, d)
    else:  # the split depends on the device's CU count
        with torch.cuda.device(device):
            nbytes = _native.lib().qim_attention_workspace_bytes(b, s, t, h, d)
    if nbytes <= 0:
        raise _native.Unsupported("attention", _native.QIM_ERR_SHAPE, f"head dim {d} (128 only)")
    return torch.empty(nbytes, device=device, dtype=torch.uint8)


def _common(name, q, k, v, ws):
    b, s, h, d = q.shape
    t = k.shape[1]
    for x, n in ((q, s), (k, t), (v, t)):
        if x is None:
            continue
        if (x.dtype != torch.bfloat16 or not x.is_cuda or x.shape != (b, n, h, d) or x.stride(3) != 1
                or x.stride(2) != d or x.stride(0) != n * x.stride(1)):
            raise _native.Unsupported(name, _native.QIM_ERR_LAYOUT,
                                      "expects bf16 (B, N, H, D) tensors with packed heads and token rows")
    if v is None and ws is None:
        raise ValueError(f"{name}: v=None needs the workspace holding V^T")
    if ws is None:
        ws = workspace(b, s, t, h, q.device, d)
    vp, ldv = (None, 0) if v is None else (_native.ptr(v), v.stride(1))
    return b, s, t, h, d, vp, ldv, ws


def attention(q, k, v, scale=None, out=None, *, workspace=None):
    """softmax(q k^T * scale) v per (batch, head): libqim's ``qim_attention``.

    q: (B, S, H, 128), k, v: (B, T, H, 128) bf16 on the GPU, each with unit
    stride inside a token and any token stride (e.g. views into a fused QKV
    projection).  scale defaults to 1/sqrt(128).  Returns (B, S, H, 128) bf16.
    ``workspace``: from ``attention.workspace`` (allocated per call if None);
    with ``v=None`` it must already hold V^T, written by the QKV projection
    (``gemm.mx_matmul_qk_norm_rope(..., vt=workspace)``, T % 64 == 0).
    The block's attention core; the reference calls torch SDPA there
    (optimizations/quantized_decode.py:70-77)."""
    b, s, t, h, d, vp, ldv, ws = _common("attention", q, k, v, workspace)
    if out is None:
        out = torch.empty((b, s, h, d), device=q.device, dtype=torch.bfloat16)
    _native.call("qim_attention", _native.ptr(q), q.stride(1), _native.ptr(k), k.stride(1), vp, ldv,
                 _native.ptr(out), out.stride(1), _native.ptr(ws), ws.numel(), b, s, t, h, d,
                 float(scale if scale is not None else d ** -0.5), _native.stream(q.device))
    return out


def attention_mxfp8(q, k, v, scale=None, *, tiled=True, out=None, workspace=None):
    """``mxfp8.quantize(attention(q, k, v).reshape(B*S, H*128), tiled=tiled)``
    in one pass (libqim's ``qim_attention_mxfp8``): the same codes and scales,
    without the bf16 output.  The block's out-projection input; the reference
    runs SDPA and then its quantize kernel (optimizations/quantized_decode.py:
    70-96).  ``out``: a preallocated ``mxfp8.empty_quantized(B*S, H*128,
    device, tiled=tiled)``; ``workspace`` and ``v=None`` as for ``attention``."""
    b, s, t, h, d, vp, ldv, ws = _common("attention_mxfp8", q, k, v, workspace)
    if out is None:
        out = mxfp8.empty_quantized(b * s, h * d, q.device, tiled=tiled)
    _native.call("qim_attention_mxfp8", _native.ptr(q), q.stride(1), _native.ptr(k), k.stride(1), vp, ldv,
                 _native.ptr(out.values), _native.ptr(out.scales), int(tiled), _native.ptr(ws), ws.numel(),
                 b, s, t, h, d, float(scale if scale is not None else d ** -0.5), _native.stream(q.device))
    return out


def qk_norm_rope(q, k, weight_q, weight_k, freqs, eps_q=1e-6, eps_k=1e-6, heads=None):
    """Fused QK-RMSNorm + RoPE without a V pack (the MMDiT block's form).

    q, k: (B, S, H, D) bf16, or (B*S, >= H*D) row views into a fused QKV
    projection output (then ``heads`` gives H and the row stride is the token
    stride).  Returns contiguous (B, S, H, D) tensors."""
    if q.ndim == 4:
        b, s, h, d = q.shape
        ldt = q.stride(1)
        if (q.stride(3) != 1 or q.stride(2) != d or k.stride() != q.stride()
                or q.stride(0) != s * q.stride(1)):
            raise _native.Unsupported("qk_norm_rope", _native.QIM_ERR_LAYOUT, "q/k layout")
    else:
        rows, width = q.shape
        h = heads
        d = width // h
        b, s = 1, rows
        ldt = q.stride(0)
        if q.stride(1) != 1 or k.stride() != q.stride():
            raise _native.Unsupported("qk_norm_rope", _native.QIM_ERR_LAYOUT, "q/k layout")
    oq = torch.empty((b, s, h, d), device=q.device, dtype=torch.bfloat16)
    ok = torch.empty_like(oq)
    f = freqs.contiguous()
    _native.call("qim_qk_norm_rope_pack", _native.ptr(q), _native.ptr(k), None, None, None,
                 _native.ptr(weight_q), _native.ptr(weight_k), _native.complex_ptr(f), _native.ptr(oq),
                 _native.ptr(ok), None, b, s, 0, h, d, ldt, float(eps_q), float(eps_k),
                 _native.stream(q.device))
    return oq, ok
