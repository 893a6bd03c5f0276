"""Plain float64 forms of attention over shared prefixes and of the 4-bit products, with bounds that count the roundings the
kernels make and no others, and inputs whose results name every key."""
import math

import torch

HALF = 2.0 ** -8    # a bf16 rounding is off by at most half a step: torch.finfo(bfloat16).eps / 2
F32 = 2.0 ** -24


def visible(s, t, n, tree):
    """(S, t + n): which keys of a prefix of t and of n own ones the S tokens see; tree over the last S own keys."""
    seen = torch.ones(s, t + n, dtype=torch.bool)
    if tree is not None:
        for j in range(s):
            if 0 <= n - s + j:
                seen[:, t + n - s + j] = tree[:, j]
    return seen


def keys_of(i, lengths, share, prefix_lengths, capacity, prefix_capacity):
    """(prefix or None, its keys, own keys) of request i, lengths clamped to what the caches hold."""
    n, p = min(max(int(lengths[i]), 0), capacity), share[i]
    if not 0 <= p < len(prefix_lengths):
        return None, 0, n
    return p, min(max(int(prefix_lengths[p]), 0), prefix_capacity), n


def attention_rows(q, k, v, seen, scale):
    """(o, bound before the output's rounding) of rows q (R, D) over keys k, v (T, D), seen (R, T), in float64.

    A key's weight: the score's 128 products are exact in fp32 and pass D + 2 additions; the factor scale * log2(e) is off by three
    roundings, its product and the difference from the row's maximum by one each, where the kernel's maximum may lag by 2^8, exp2 by
    one unit (2 F32).  Moves of the maximum multiply what was summed by powers of 2 whose exponents add up to the scores' range: at most one
    move for every block of 32 keys and every join of a piece.  What all weights of a row share cancels.  Numerator: p enters the product
    as two bf16 terms (2^-16 of it is left), its sum passes two matrix instructions of 32 for a block and the joins;
    denominator: one addition for a block; then a reciprocal and a product."""
    d, t = q.shape[1], k.shape[0]
    w = q @ k.T * scale
    w = w.masked_fill(~seen, -math.inf)
    top = w.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(w - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    v = torch.where(seen.any(0)[:, None], v, torch.zeros_like(v))
    o, mag = p @ v, p @ v.abs()
    depth = (top - w).masked_fill(~seen, 0)
    steps = t / 32 + 64
    dx = F32 * ((d + 2) * scale * (q.abs() @ k.abs().T) + 4 * w.masked_fill(~seen, 0).abs() + 2 * depth + depth.amax(-1, keepdim=True) + 16 + 3 * steps)
    px = p * dx
    bound = px @ v.abs() + o.abs() * px.sum(-1, keepdim=True) + (2.0 ** -16 + (64 + 2 * steps) * F32) * mag + (16 + steps) * F32 * o.abs()
    return o, 1.01 * bound


def attention_shared(q, prefix, cache, lengths, share, prefix_lengths, tree=None, scale=None):
    """(o, bound): prefix and cache are (K, V) values, share a list; as attention.attention_shared defines it."""
    q = q.double().cpu()
    pk, pv, ck, cv = (t.double().cpu() for t in (*prefix, *cache))
    b, s, h, d = q.shape
    hk = ck.shape[2]
    g = h // hk
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(b):
        p, t, n = keys_of(i, lengths, share, prefix_lengths, ck.shape[1], pk.shape[1])
        seen = visible(s, t, n, None if tree is None else (tree if tree.dim() == 2 else tree[i]).cpu())
        if t + n == 0:
            continue
        for j in range(hk):
            k, v = ck[i, :n, j], cv[i, :n, j]
            if t:
                k, v = torch.cat([pk[p, :t, j], k]), torch.cat([pv[p, :t, j], v])
            rows = q[i, :, j * g:(j + 1) * g].reshape(s * g, d)
            o, e = attention_rows(rows, k, v, seen.repeat_interleave(g, 0), d ** -0.5 if scale is None else scale)
            out[i, :, j * g:(j + 1) * g], bound[i, :, j * g:(j + 1) * g] = o.view(s, g, d), e.view(s, g, d)
    return out, bound


def rounded(y, e, dtype=torch.bfloat16):
    """The bound of a result whose exact value is y, off by e before its rounding to dtype."""
    return e + (HALF if dtype == torch.bfloat16 else F32) * (y.abs() + e) + 2.0 ** -133


def four_bit(x, codes, scales, zeros):
    """(y, error before the output's rounding) in float64 of x (M, K) times an unpacked 4-bit weight.

    The weights enter exactly (q - z has 4 significand bits, E2M1 times a power of two too), so do the products; a term passes the 32
    additions of its matrix instruction, one for each later step of the chain (at most K / 32), its group's scaling and addition
    (2) and a join of up to 16 partial sums: that many F32 of |x| |w|."""
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(1).cpu()
    group = x.shape[1] // scales.shape[1]
    if scales.dtype == torch.uint8:
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
        w = torch.where(q >= 8, -1.0, 1.0) * table[q.long() & 7] * torch.exp2(scales.cpu().double() - 127).repeat_interleave(group, 1)
    else:
        z = (torch.full_like(scales, 8) if zeros is None else zeros).cpu().double().repeat_interleave(group, 1)
        w = (q.double() - z) * scales.cpu().double().repeat_interleave(group, 1)
    x = x.double().cpu()
    return x @ w.T, (32 + x.shape[1] / 32 + 20) * F32 * (x.abs() @ w.abs().T)


# ---- values that name their keys

def counted(g, lead, keys, d=128):
    """(*lead, keys, d) of 0 and 1, one 1 to a key: every one of the d places equally often (one more for the first keys' rest),
    in any order.  With equal weights a row's output counts the keys: one skipped or taken twice moves a place by 1 in keys / d."""
    v = torch.zeros(*lead, keys, d)
    flat = v.view(-1, keys, d)
    for i in range(flat.shape[0]):
        flat[i, torch.arange(keys), torch.randperm(keys, generator=g) % d] = 1
    return v


def signs(g, shape):
    """Values of +1 and -1: 16 times one of them, against itself, scores 181 over sqrt(128), and some 16 in deviation against others."""
    return torch.randint(0, 2, shape, generator=g).float() * 2 - 1


def edges(t):
    """Keys of a length of t: its ends, those beside every multiple of 32, and a spread of others."""
    near = [k + j for k in range(0, t + 1, 32) for j in (-1, 0, 1)]
    return sorted({k for k in near + list(range(0, t, 7)) + [t - 1] if 0 <= k < t})
