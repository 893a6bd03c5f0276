"""Products of a few rows with 4-bit weights.

Half a byte a weight where ``MXFP8Linear`` holds one, and the activation in
bf16: for projections of a few tokens, whose time is the weight's bytes.  Two
kinds of weight (the reference has neither; there is no reference
counterpart):

    int4    s (q - z): codes q 0..15, a bf16 scale s and optionally a zero point z 0..15 (else 8)
            for each group of 32, 64 or 128 values of a row
    mxfp4   an E2M1 number times 2^(e - 127), an E8M0 exponent e for 32 values of a row

``pack_weight`` lays the codes of a checkpoint out once, ``quantize_weight`` makes
them from a bf16 weight; ``matmul`` and ``swiglu`` are the products (libqim's
``qim_fourbit_matmul``).
"""
from typing import NamedTuple, Optional

import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels.adapters import row_layout

KINDS = ("int4", "mxfp4")
GROUPS = (32, 64, 128)
MX_GROUP = 32
TILE, STEP = 16, 128   # rows of a weight tile, values of k of a step
MAX_STRIDE = 1 << 24   # elements between rows of x that the kernels take


class FourBitWeight(NamedTuple):
    """A weight (N, K) in the kernels' layout: rows in tiles of 16, k in steps of 128 (the last of each padded)."""

    codes: torch.Tensor             # (tiles, steps, 64, 16) uint8: 16 bytes of each lane
    scales: torch.Tensor            # int4: (tiles, steps, 4, 128 / group, 4) bf16, row 4 a + c of a tile at (a, :, c); mxfp4:
                                    # (tiles, steps, 16, 4) uint8
    zeros: Optional[torch.Tensor]   # int4: (tiles, steps, 16, 128 / group) uint8, or None
    rows: int                       # N
    width: int                      # K
    group: int                      # 32, 64 or 128

    @property
    def kind(self):
        return "mxfp4" if self.scales.dtype == torch.uint8 else "int4"


def _padded(t, rows, width):
    """t (R, W) with zeros up to (rows, width)."""
    return torch.nn.functional.pad(t, (0, width - t.shape[1], 0, rows - t.shape[0]))


def pack_weight(codes, scales, *, zeros=None):
    """A ``FourBitWeight`` from a checkpoint's: codes (N, K / 2) uint8, two to a byte, the first in the low half;
    scales (N, K / group), bf16 for int4, uint8 (or float8_e8m0fnu) for mxfp4 with its groups of 32; zeros (N, K / group) uint8
    0..15, or None.  On any device; the result is on the same."""
    if scales.dtype == torch.float8_e8m0fnu:
        scales = scales.view(torch.uint8)
    if codes.dim() != 2 or scales.dim() != 2 or codes.dtype != torch.uint8 or scales.dtype not in (torch.bfloat16, torch.uint8):
        raise ValueError("codes is a (N, K / 2) uint8 tensor, scales a (N, K / group) bf16 (int4) or uint8 (mxfp4) one")
    n, k = codes.shape[0], 2 * codes.shape[1]
    mx = scales.dtype == torch.uint8
    if n == 0 or k == 0 or scales.shape[0] != n or scales.shape[1] == 0 or k % scales.shape[1]:
        raise ValueError(f"scales {tuple(scales.shape)} of codes {tuple(codes.shape)}")
    group = k // scales.shape[1]
    if group not in ((MX_GROUP,) if mx else GROUPS):
        raise ValueError(f"groups of {group}: {MX_GROUP} for mxfp4, one of {GROUPS} for int4")
    if zeros is not None and (mx or zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
        raise ValueError("zeros is a uint8 tensor of the scales' shape, for int4")
    if mx and int(scales.max()) == 255:
        raise ValueError("an exponent of 255 (NaN)")
    if zeros is not None and int(zeros.max()) > 15:
        raise ValueError("a zero point is 0 to 15")
    if len({t.device for t in (codes, scales, zeros) if t is not None}) > 1:
        raise ValueError("codes, scales and zeros are on one device")
    tiles, steps = (n + TILE - 1) // TILE, (k + STEP - 1) // STEP
    c = _padded(codes, tiles * TILE, steps * STEP // 2)
    if not mx:  # byte i of a lane's 8 codes: code i low, code i + 4 high
        c = torch.stack([c & 15, c >> 4], dim=-1).view(-1, 2, 4)
        c = c[:, 0] | c[:, 1] << 4
    # (tile, n, step, j, kg, 4 bytes) -> (tile, step, kg, n, j, 4 bytes)
    c = c.reshape(tiles, TILE, steps, 4, 4, 4).permute(0, 2, 4, 1, 3, 5).reshape(tiles, steps, 64, 16).contiguous()
    per = STEP // group

    def by_step(t):
        return _padded(t, tiles * TILE, steps * per).view(tiles, TILE, steps, per).permute(0, 2, 1, 3).contiguous()
    s = by_step(scales)
    if not mx:
        s = s.view(tiles, steps, 4, 4, per).transpose(3, 4).contiguous()
    return FourBitWeight(c, s, None if zeros is None else by_step(zeros), n, k, group)


def unpack_weight(weight):
    """(codes, scales, zeros) as ``pack_weight`` takes them."""
    tiles, steps = weight.codes.shape[:2]
    n, k, per = weight.rows, weight.width, STEP // weight.group
    mx = weight.kind == "mxfp4"
    c = weight.codes.view(tiles, steps, 4, TILE, 4, 4).permute(0, 3, 1, 4, 2, 5).reshape(tiles * TILE, steps * STEP // 2)
    if not mx:
        c = c.reshape(-1, 4)
        c = torch.cat([c & 15, c >> 4], dim=-1)
        c = (c[:, 0::2] | c[:, 1::2] << 4).view(tiles * TILE, steps * STEP // 2)

    def by_row(t):
        return t.permute(0, 2, 1, 3).reshape(tiles * TILE, steps * per)[:n, :k // weight.group].contiguous()
    s = weight.scales if mx else weight.scales.transpose(3, 4).reshape(tiles, steps, TILE, per)
    return c[:n, :k // 2].contiguous(), by_row(s), None if weight.zeros is None else by_row(weight.zeros)


E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def dequantize_weight(weight):
    """The fp32 (N, K) weight that the codes stand for (exact)."""
    codes, scales, zeros = unpack_weight(weight)
    q = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(1)
    if weight.kind == "mxfp4":
        table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=q.device)
        return torch.ldexp(table[q.int()].unflatten(1, (-1, MX_GROUP)), (scales.int() - 127).unsqueeze(-1)).flatten(1)
    z = 8.0 if zeros is None else zeros.float().unsqueeze(-1)
    return ((q.float().unflatten(1, (-1, weight.group)) - z) * scales.float().unsqueeze(-1)).flatten(1)


def quantize_weight(w, kind="int4", group=64, *, symmetric=False):
    """A ``FourBitWeight`` of a weight (N, K), K a multiple of the group (32 for mxfp4), every code the nearest.

    int4: the scale is a group's span / 15 with a zero point, or with ``symmetric`` its largest magnitude / 7; rounded to
    bf16 before the codes are taken.  mxfp4: the exponent that brings the largest magnitude to 4..8 (then at most 6), as the
    OCP MX formats define it, or the next one where that is nearer in squares.  A weight that holds infinities or NaN, in fp32, is refused."""
    if kind not in KINDS:
        raise ValueError(f"kind {kind!r}: int4 or mxfp4")
    group = MX_GROUP if kind == "mxfp4" else group
    if group not in GROUPS or w.dim() != 2 or w.shape[0] == 0 or w.shape[1] == 0 or w.shape[1] % group:
        raise ValueError(f"a weight {tuple(w.shape)} in groups of {group}: (N, K), K a multiple of one of {GROUPS}")
    w = w.detach().float()
    if not torch.isfinite(w).all():
        raise ValueError("the weight holds infinities, NaN or values that fp32 does not")
    g = w.unflatten(1, (-1, group))
    zeros = None
    if kind == "mxfp4":
        edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
        table = torch.tensor(E2M1, device=w.device)
        top = g.abs().amax(-1, keepdim=True)
        first = (torch.frexp(top)[1] - 3).clamp(-127, 127)
        best = None
        for e in (first, (first + 1).clamp(max=127)):
            y = torch.ldexp(g, -e)
            q = torch.bucketize(y.abs(), edges)
            err = (torch.ldexp(table[q], e) - g.abs()).square().sum(-1, keepdim=True)
            if best is None:
                best = (err, e, q)
            else:
                take = err < best[0]
                best = (err, torch.where(take, e, best[1]), torch.where(take, q, best[2]))
        _, e, q = best
        q, scales = q + 8 * (g < 0), (e + 127).squeeze(-1).to(torch.uint8)
    elif symmetric:
        scales = (g.abs().amax(-1) / 7).to(torch.bfloat16)
        s = scales.float().unsqueeze(-1)
        q = torch.where(s > 0, torch.round(g / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(g)).clamp(-8, 7) + 8
    else:
        lo, hi = g.amin(-1, keepdim=True).clamp(max=0), g.amax(-1, keepdim=True).clamp(min=0)
        scales = (hi / 15 - lo / 15).squeeze(-1).to(torch.bfloat16)   # (the span itself may pass fp32's range)
        s = scales.float().unsqueeze(-1)
        s = torch.where(s > 0, s, torch.ones_like(s))
        z = torch.round(-lo / s).clamp(0, 15)
        q, zeros = (torch.round(g / s) + z).clamp(0, 15), z.squeeze(-1).to(torch.uint8)
    q = q.to(torch.uint8).flatten(1)
    return pack_weight(q[:, 0::2] | q[:, 1::2] << 4, scales, zeros=zeros)


def _check_weight(name, w, device):
    """The addresses of a weight's tensors, checked against its sizes."""
    tiles, steps, per = (w.rows + TILE - 1) // TILE, (w.width + STEP - 1) // STEP, STEP // w.group if w.group in GROUPS else 0
    by_row = (tiles, steps, TILE, per)
    shape = by_row if w.scales.dtype == torch.uint8 else (tiles, steps, 4, per, 4)
    if not (per and w.rows > 0 and w.width > 0 and w.codes.shape == (tiles, steps, 64, 16) and w.codes.dtype == torch.uint8
            and w.scales.shape == shape and (w.scales.dtype == torch.bfloat16 or w.scales.dtype == torch.uint8 and w.group == MX_GROUP)
            and (w.zeros is None or (w.zeros.shape == by_row and w.zeros.dtype == torch.uint8 and w.scales.dtype == torch.bfloat16))
            and all(t is None or (t.device == device and t.is_contiguous()) for t in w[:3])):
        raise _native.Unsupported(name, _native.QIM_ERR_LAYOUT, f"expects a FourBitWeight of pack_weight or quantize_weight on {device}")
    return w.codes.data_ptr(), w.scales.data_ptr(), _native.ptr(w.zeros)


def _product(name, x, first, second, bias, out, dtype):
    def refuse(why):
        raise _native.Unsupported(name, _native.QIM_ERR_LAYOUT, why)
    device = x.device
    if not x.is_cuda:
        refuse("expects tensors on the GPU")
    lay = row_layout(x) if x.dtype == torch.bfloat16 else None
    if lay is None or lay[1] != first.width:
        refuse(f"x is a bf16 (M, {first.width}) or (B, S, {first.width}) tensor with rows one stride apart")
    if lay[2] >= MAX_STRIDE:   # (a token of each of several long sequences; the kernels' offsets within a tile are 32-bit)
        x = x.contiguous()
        lay = row_layout(x)
    weights = _check_weight(name, first, device)
    if second is None:
        weights += (None, None, None)
    else:
        if (second.rows, second.width, second.group, second.kind, second.zeros is None) != (
                first.rows, first.width, first.group, first.kind, first.zeros is None):
            refuse("gate and up are weights of one shape and kind")
        weights += _check_weight(name, second, device)
    n = first.rows
    if dtype not in (torch.bfloat16, torch.float32):
        refuse(f"an output of {dtype}: bf16 or fp32")
    if bias is not None and (bias.dtype != torch.bfloat16 or bias.shape != (n,) or bias.device != device or not bias.is_contiguous()):
        refuse(f"bias is a contiguous bf16 ({n},) tensor on {device}")
    shape = x.shape[:-1] + (n,)
    if out is None:
        out, ldo = x.new_empty(shape, dtype=dtype), n
    else:
        o = row_layout(out) if out.dtype == dtype and out.shape == shape and out.device == device else None
        if o is None:
            refuse(f"out is a {dtype} {tuple(shape)} tensor on {device} with rows one stride apart")
        ldo = o[2]
    if lay[0] == 0:
        return out
    _native.call_on(device, "qim_fourbit_matmul", x.data_ptr(), lay[2], 0 if first.kind == "mxfp4" else first.group, *weights,
                    _native.ptr(bias), out.data_ptr(), ldo, int(dtype == torch.float32), lay[0], n, first.width)
    return out


def matmul(x, weight, *, bias=None, out=None, dtype=torch.bfloat16):
    """``x @ W.T (+ bias)``: x (M, K) or (B, S, K) bf16 on the GPU, rows any multiple of 8 elements apart (copied
    if 2^24 or more); W a ``FourBitWeight`` (N, K); bias bf16 (N,).  Returns (..., N) of ``dtype`` (bf16 or fp32), in ``out`` if
    given (any row stride, apart from x, weight and bias).  The weights enter exactly, sums are fp32, the result is rounded
    once.  Meant for up to some hundred rows; it takes fewer than 2^20, and fewer than some 4 * 10^10 values of output (half as
    many with ``swiglu``).  No gradient is recorded."""
    return _product("fourbit.matmul", x, weight, None, bias, out, dtype)


def swiglu(x, gate, up, *, out=None, dtype=torch.bfloat16):
    """``silu(x @ gate.T) * (x @ up.T)`` in one launch, rounded once: two weights of one shape and kind, the rest as in
    ``matmul``."""
    return _product("fourbit.swiglu", x, gate, up, None, out, dtype)
