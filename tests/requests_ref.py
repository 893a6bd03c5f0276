"""Plain float64 forms of the many-request operators (MXFP8 K/V cache, attention
over it, low-rank adapters) and the error bounds their tests use."""
import math

import torch

HALF = 2.0 ** -8    # a bf16 rounding is off by at most half a step: torch.finfo(bfloat16).eps / 2
F32 = 2.0 ** -24


def block_values(x):
    """The float64 values of x (..., D) held in MXFP8: per 32 values the smallest power of two
    2^(e - 127), 0 <= e <= 254, that brings the largest magnitude to at most 448, and per value the nearest
    E4M3 number (ties to even).  Finite x."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    mant, exp = torch.frexp(top)
    e = (exp - 9 + (mant > 0.875).to(exp.dtype)).clamp(-127, 127).double()
    unit = torch.where(top > 0, torch.exp2(e), torch.full_like(e, 2.0 ** -127))
    y = g / unit
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(y / step) * step * unit).flatten(-2)


def attention(q, k, v, lengths, tree=None, scale=None):
    """(o, bound) in float64 on the CPU: q (B, S, H, D), k, v (B, C, HK, D) values, lengths (B,).

    The bound: p is rounded to bf16 for the product with V (HALF of each term), a score of D products
    in fp32 is off by at most D * F32 * sum |q k| (and 2 more roundings), which moves p by that much relative
    to its size, in the numerator and in the sum; exp2 and the join of partial sums add a few F32 (64 are
    allowed); the output is rounded once."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    b, s, h, d = q.shape
    g = h // k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out, bound = torch.zeros(b, s, h, d, dtype=torch.float64), torch.zeros(b, s, h, d, dtype=torch.float64)
    for i in range(b):
        n = min(max(int(lengths[i]), 0), k.shape[1])
        if n == 0:
            continue
        seen = torch.ones(s, n, dtype=torch.bool)
        if tree is not None:
            m = (tree if tree.dim() == 2 else tree[i]).cpu()
            first = max(0, s - n)
            seen[:, n - (s - first):] = m[:, first:]
        for j in range(h):
            kk, vv = k[i, :n, j // g], v[i, :n, j // g]
            w = (q[i, :, j] @ kk.T * scale).masked_fill(~seen, -math.inf)
            top = w.amax(-1, keepdim=True)
            p = torch.exp(w - torch.where(top == -math.inf, torch.zeros_like(top), top))
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total == 0, torch.ones_like(total), total)
            # A key that a row does not see adds nothing to it, whatever it holds.
            pv = torch.stack([p[r, seen[r]] @ vv[seen[r]] for r in range(s)])
            mag = torch.stack([p[r, seen[r]] @ vv[seen[r]].abs() for r in range(s)])
            ds = ((d + 2) * F32 * scale * (q[i, :, j].abs() @ kk.abs().T)).masked_fill(~seen, 0).amax(-1, keepdim=True)
            out[i, :, j] = pv
            bound[i, :, j] = (HALF + 4 * ds + 64 * F32) * mag + HALF * pv.abs()
    return out, bound


def low_rank(x, down, up, index, scale=None, base=None, parts=1):
    """(y, bound) in float64: x (M, K), index (M,).

    The bound: each of the K products of h in fp32 adds at most F32 of the sum of magnitudes per addition
    (K + 16 of them, the join of chunks among them); h enters the second product as two bf16 terms, off by at most
    HALF^2 of it; R + 2 fp32 additions there, two of them twice as long (hi and lo); scale and base add two roundings; the
    result is rounded once."""
    m, k = x.shape
    a, n, r = up.shape
    x64, d64, u64 = x.double(), down.double(), up.double()
    y = torch.zeros(m, n, dtype=torch.float64, device=x.device) if base is None else base.double().clone()
    mag = y.abs() * 2 * F32
    w = n // parts
    for i in range(a):
        rows = (index == i).nonzero()[:, 0]
        if not len(rows):
            continue
        sc = 1.0 if scale is None else float(scale[i])
        for j in range(parts):
            dn, u = d64[i, j * r:(j + 1) * r], u64[i, j * w:(j + 1) * w]
            h, hm = x64[rows] @ dn.T, x64[rows].abs() @ dn.abs().T
            cols = slice(j * w, (j + 1) * w)
            y[rows, cols] += sc * (h @ u.T)
            eh = (k + 16) * F32 * hm + HALF * HALF * h.abs()
            mag[rows, cols] += abs(sc) * (eh @ u.abs().T + (2 * r + 8) * F32 * (h.abs() @ u.abs().T))
    return y, mag + HALF * (y.abs() + mag)
