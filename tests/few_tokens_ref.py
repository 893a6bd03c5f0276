"""Plain float64 forms of the operators of a step of a few tokens (residual with norms, 4-bit weights, attention
over shared prefixes) and the error bounds their tests use."""
import math

import torch

HALF = 2.0 ** -8    # a bf16 rounding is off by at most half a step: torch.finfo(bfloat16).eps / 2
F32 = 2.0 ** -24


def _normed(y, e, norm):
    """(n, error) of a norm of y (..., D) whose values are off by at most e: kind, weight, eps.

    A shift of y by e moves the mean by at most mean(e), the deviation's square root by at most sqrt(mean(e^2)) (the
    triangle inequality), relative to it times rstd; the sums are float64, the mean two fp32 terms, the variance
    and its root one fp32 rounding each, and four multiplications and subtractions follow."""
    kind, w, eps = norm
    d = y.shape[-1]
    mean = y.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(y[..., :1])
    emean = e.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(mean)
    r = 1 / torch.sqrt((y - mean).square().sum(-1, keepdim=True) / d + eps)
    n = (y - mean) * r
    en = (e + emean) * r + n.abs() * ((e + emean).square().mean(-1, keepdim=True).sqrt() * r + 8 * F32)
    if w is None:
        return n, en
    w = w.double().cpu()
    return n * w, en * w.abs() + F32 * (n * w).abs()


def residual_norm(h, x, norm, gate=None, alpha=1.0, post=None, scale=None, shift=None, add_one=False):
    """(h', bound, z, bound before z's own rounding) in float64 on the CPU.  norm, post: (kind, weight, eps) or None."""
    h, x = h.double().cpu(), x.double().cpu()
    u, e = x, torch.zeros_like(x)
    if post is not None:
        u, e = _normed(u, e, post)
    if gate is not None:
        g = gate.double().cpu()
        u, e = u * g, e * g.abs() + F32 * (u * g).abs()
    hs = h + alpha * u
    eh = abs(alpha) * e + F32 * (hs.abs() + 2 * abs(alpha) * u.abs())
    z, ez = _normed(hs, eh, norm)
    if scale is not None:
        s = scale.double().cpu() + (1.0 if add_one else 0.0)
        z, ez = z * s, ez * s.abs() + 2 * F32 * (z * s).abs()
    if shift is not None:
        z = z + shift.double().cpu()
        ez = ez + F32 * z.abs()
    return hs, eh + HALF * (hs.abs() + eh), z, ez


def four_bit(x, codes, scales, zeros, bias=None):
    """(y, error before the output's rounding) in float64 of x (M, K) with an unpacked weight.

    Products of bf16 values with codes are exact in fp32.  A term passes the additions of its matrix
    instruction (32), one for each later step of the chain (at most K / 32), a join of up to 16 partial sums, and for int4 the
    scale and zero point (4): that many F32 of the magnitudes, where int4 sums q x and z x apart."""
    k = x.shape[1]
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(1).cpu().double()
    group = k // scales.shape[1]
    x = x.double().cpu()
    if scales.dtype == torch.uint8:
        mag = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
        c = q.long()
        unit = torch.exp2(scales.cpu().double() - 127).repeat_interleave(group, 1)
        w = torch.where(c >= 8, -1.0, 1.0) * mag[c & 7] * unit
        big = w.abs()
    else:
        s = scales.cpu().double().repeat_interleave(group, 1)
        z = (torch.full_like(scales, 8) if zeros is None else zeros).cpu().double().repeat_interleave(group, 1)
        w, big = (q - z) * s, (q + z) * s.abs()
    y, e = x @ w.T, (32 + k / 32 + 20) * F32 * (x.abs() @ big.T)
    if bias is not None:
        y = y + bias.cpu().double()
        e = e + F32 * y.abs()
    return y, e


def swiglu(gate, up):
    """(y, error) of silu(g) * u from (value, error) pairs.  |silu'| < 1.1; e^-g is off by |g| F32 from its argument
    and a few F32 from the instruction, where it is not negligible beside fp32's range (2^-120)."""
    g, eg = gate
    u, eu = up
    s = g * torch.sigmoid(g)
    es = 1.1 * eg + (g.abs() + 8) * F32 * s.abs() + 2.0 ** -120
    return s * u, es * u.abs() + (s.abs() + es) * eu + F32 * (s * u).abs()


def rounded(y, e, dtype=torch.bfloat16):
    """The bound of a result whose exact value is y, off by e before its rounding to dtype."""
    return e + (HALF if dtype == torch.bfloat16 else F32) * (y.abs() + e) + 2.0 ** -133


def attention_shared(q, prefix, cache, lengths, share, prefix_lengths, tree=None, scale=None):
    """(o, bound) in float64 on the CPU: prefix and cache are (K, V) values, share a list (one prefix or -1 per
    sequence).  The bound as requests_ref.attention derives it, over the keys of both."""
    q = q.double().cpu()
    pk, pv, ck, cv = (t.double().cpu() for t in (*prefix, *cache))
    b, s, h, d = q.shape
    g = h // ck.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out, bound = torch.zeros(b, s, h, d, dtype=torch.float64), torch.zeros(b, s, h, d, dtype=torch.float64)
    for i in range(b):
        n = min(max(int(lengths[i]), 0), ck.shape[1])
        p = share[i]
        t = min(max(int(prefix_lengths[p]), 0), pk.shape[1]) if 0 <= p < pk.shape[0] else 0
        seen = torch.ones(s, t + n, dtype=torch.bool)
        if tree is not None:
            m = (tree if tree.dim() == 2 else tree[i]).cpu()
            first = max(0, s - n)
            seen[:, t + n - (s - first):] = m[:, first:]
        if t + n == 0:
            continue
        for j in range(h):
            k, v = ck[i, :n, j // g], cv[i, :n, j // g]
            if t:
                k, v = torch.cat([pk[p, :t, j // g], k]), torch.cat([pv[p, :t, j // g], v])
            w = (q[i, :, j] @ k.T * scale).masked_fill(~seen, -math.inf)
            top = w.amax(-1, keepdim=True)
            e = torch.exp(w - torch.where(top == -math.inf, torch.zeros_like(top), top))
            total = e.sum(-1, keepdim=True)
            e = e / torch.where(total == 0, torch.ones_like(total), total)
            o = torch.stack([e[r, seen[r]] @ v[seen[r]] for r in range(s)])
            mag = torch.stack([e[r, seen[r]] @ v[seen[r]].abs() for r in range(s)])
            ds = ((d + 2) * F32 * scale * (q[i, :, j].abs() @ k.abs().T)).masked_fill(~seen, 0).amax(-1, keepdim=True)
            out[i, :, j] = o
            bound[i, :, j] = (HALF + 4 * ds + 64 * F32) * mag + HALF * o.abs()
    return out, bound
