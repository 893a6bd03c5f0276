"""Performance cases of the operators of a step of a few tokens: the residual with the norms around it,
products of few rows with 4-bit weights, and attention of many requests that continue shared prefixes.

Sizes are those of the repository's configurations: hidden 4096 with 32 heads of 128, FFN 12288, images of 1024
tokens, prefixes of a 512^2 image and its text (1101 tokens) up to two edited images (8392), and generic ones where
those say nothing (shared K/V heads, long prefixes, groups of weights).

With ``own`` false an operator is computed in plain torch operations in float32, rounded once at its end;
``exact`` restates the definitions in float64, apart from that.
"""
import math
import os
import random
import sys
import types

import torch

own = False

HEAD = 128
EPS = 1e-6
PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-image-2.1-accel_amd")


def listed():
    return [
        # One new token of each of 16 requests between two RMS norms: latency.
        {"name": "norm_tokens", "op": "norm", "batch": 16, "seq": 1, "dim": 4096, "post": "rms", "norm": "rms",
         "modulated": False},
        # The block's own form at 512^2, two requests: gated residual, LayerNorm, scale and shift.
        {"name": "norm_512", "op": "norm", "batch": 2, "seq": 1024, "dim": 4096, "post": "none", "norm": "layer",
         "modulated": True},
        # A 2048^2 image, a norm on both sides of the block and every modulation.
        {"name": "norm_2048", "op": "norm", "batch": 1, "seq": 16384, "dim": 4096, "post": "rms", "norm": "rms",
         "modulated": True},
        # One token of one request through an up projection: latency, 25 MB of weights.
        {"name": "four_token", "op": "four", "rows": 1, "k": 4096, "n": 12288, "kind": "int4", "group": 128,
         "zeros": False, "bias": False, "swiglu": False},
        # One token of each of 16 requests through the down projection, codes of the MX family, a bias.
        {"name": "four_down", "op": "four", "rows": 16, "k": 12288, "n": 4096, "kind": "mxfp4", "group": 32,
         "zeros": False, "bias": True, "swiglu": False},
        # 24 drafted tokens through gate and up projections and the SwiGLU.
        {"name": "four_swiglu", "op": "four", "rows": 24, "k": 4096, "n": 12288, "kind": "int4", "group": 64,
         "zeros": True, "bias": False, "swiglu": True},
        # The text tokens of two prompts through the stacked Q/K/V projection.
        {"name": "four_prompts", "op": "four", "rows": 154, "k": 4096, "n": 12288, "kind": "int4", "group": 32,
         "zeros": True, "bias": False, "swiglu": False},
        # The largest number of rows that these weights are meant for: a 512^2 image.
        {"name": "four_image", "op": "four", "rows": 1024, "k": 4096, "n": 4096, "kind": "mxfp4", "group": 32,
         "zeros": False, "bias": False, "swiglu": False},
        # Four variants of one request, a token each: latency.
        {"name": "share_token", "op": "share", "batch": 4, "seq": 1, "prefixes": 1, "prefix": 1101, "capacity": 96,
         "heads": 32, "kv_heads": 32, "tree": False},
        # 32 requests over one editing prefix, 4 query heads to a K/V head.
        {"name": "share_batch", "op": "share", "batch": 32, "seq": 1, "prefixes": 1, "prefix": 8392, "capacity": 1024,
         "heads": 32, "kv_heads": 8, "tree": False},
        # 24 drafted tokens of each of 8 requests, a tree per request.
        {"name": "share_tree", "op": "share", "batch": 8, "seq": 24, "prefixes": 1, "prefix": 8392, "capacity": 256,
         "heads": 32, "kv_heads": 32, "tree": True},
        # 48 requests on 5 long prefixes of different lengths, some requests on none.
        {"name": "share_groups", "op": "share", "batch": 48, "seq": 1, "prefixes": 5, "prefix": 32768, "capacity": 640,
         "heads": 32, "kv_heads": 8, "tree": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "four", "four", "share", "share"))
    if op == "norm":
        dim = 8 * _log(rng, 32, 1024)
        rows = _log(rng, 1, 16384 * 4096 // max(dim, 4096))
        batch = rng.randint(1, min(rows, 32))
        return {"op": op, "batch": batch, "seq": rows // batch, "dim": dim, "post": rng.choice(("none", "rms", "layer")),
                "norm": rng.choice(("rms", "layer")), "modulated": rng.random() < 0.6}
    if op == "four":
        kind = rng.choice(("int4", "int4", "mxfp4"))
        group = rng.choice((32, 64, 128)) if kind == "int4" else 32
        rows = _log(rng, 1, 1024)
        k = group * _log(rng, max(2, 512 // group), 12288 // group)
        n = min(_log(rng, 96, 16384), 12288 * 4096 // k, max(96, 1024 * 4096 * 4096 // (k * rows)))
        return {"op": op, "rows": rows, "k": k, "n": n, "kind": kind, "group": group,
                "zeros": kind == "int4" and rng.random() < 0.6, "bias": rng.random() < 0.3, "swiglu": rng.random() < 0.3}
    kv = rng.choice((4, 8, 16, 32))
    heads = kv * rng.choice((1, 2, 4)) if kv < 32 else kv
    batch, seq, prefixes = _log(rng, 1, 64), rng.choice((1, 1, 1, 2, 5, 16, 33, 64)), rng.choice((1, 1, 1, 2, 3, 6))
    most = min(32768, 65536 * 8 // (prefixes * kv), 32768 * 64 * 32 // (batch * seq * heads))
    capacity = min(seq + _log(rng, 1, 1024), max(seq, 32 * 1024 * 8 // (batch * kv)))
    return {"op": op, "batch": batch, "seq": seq, "prefixes": prefixes, "prefix": _log(rng, 16, max(64, most)),
            "capacity": capacity, "heads": heads, "kv_heads": kv, "tree": seq > 1 and rng.random() < 0.7}


# ------------------------------------------------------------------ inputs --

def _share(case):
    """The prefix that each request continues; of several prefixes a few requests have none (-1)."""
    if case["prefixes"] == 1:
        return [0] * case["batch"]
    r = random.Random(case["batch"] * 31 + case["prefix"])
    return [-1 if r.random() < 0.1 else r.randrange(case["prefixes"]) for _ in range(case["batch"])]


def _prefix_lengths(case):
    """Valid keys of each prefix: the longest first, down to about half of it."""
    t, n = case["prefix"], case["prefixes"]
    return [max(1, t - t * i // (2 * n)) for i in range(n)]


def _lengths(case):
    """Own keys of each request, its new tokens among them."""
    b, c, s = case["batch"], case["capacity"], case["seq"]
    return [max(s, c - (c - s) * i // b) for i in range(b)]


def _quantized(x):
    """x (..., D) -> E4M3 codes and E8M0 exponents (bytes), one per 32 values: the smallest power of two that brings the
    largest magnitude to at most 448."""
    blocks = x.float().unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1)
    mantissa, exponent = torch.frexp(top)                      # top = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - 1 - 8 + (mantissa > 0.875).to(exponent.dtype) + 127
    e = torch.where(top == 0, torch.zeros_like(e), e.clamp(0, 254))
    codes = torch.ldexp(blocks, (127 - e).unsqueeze(-1)).to(torch.float8_e4m3fn).flatten(-2)
    return codes, e.to(torch.uint8)


def _values(codes, exponents):
    """The float32 values that codes (..., D) and exponents (..., D/32) stand for."""
    return torch.ldexp(codes.float().unflatten(-1, (-1, 32)), exponents.int().unsqueeze(-1) - 127).flatten(-2)


def _tree(b, s, seed):
    """(B, S, S) truth values: drafted token i sees itself and its ancestors, each parent earlier than its child."""
    r = random.Random(seed)
    m = torch.zeros(b, s, s, dtype=torch.bool)
    for i in range(b):
        for j in range(s):
            if j:
                m[i, j] = m[i, r.randrange(max(0, j - 8), j)]
            m[i, j, j] = True
    return m


def _four_bits(w, case):
    """A weight (N, K) as a checkpoint holds it: codes (N, K / 2), two to a byte, the first in the low half; scales
    (N, K / group), bf16 for int4 and E8M0 bytes for mxfp4; zero points (N, K / group) bytes or None."""
    g = w.float().unflatten(-1, (-1, case["group"]))
    zeros = None
    if case["kind"] == "mxfp4":
        top = g.abs().amax(-1).clamp(min=1e-30)
        scales = (torch.floor(torch.log2(top)) - 2 + 127).to(torch.uint8)
        y = g / torch.exp2(scales.float() - 127).unsqueeze(-1)
        edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
        q = torch.bucketize(y.abs(), edges) + 8 * (y < 0)
    elif case["zeros"]:
        lo, hi = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
        scales = ((hi - lo).clamp(min=1e-6) / 15).to(torch.bfloat16)
        zeros = torch.round(-lo / scales.float()).clamp(0, 15).to(torch.uint8)
        q = torch.round(g / scales.float().unsqueeze(-1) + zeros.float().unsqueeze(-1)).clamp(0, 15)
    else:
        scales = (g.abs().amax(-1).clamp(min=1e-6) / 7).to(torch.bfloat16)
        q = torch.round(g / scales.float().unsqueeze(-1)).clamp(-8, 7) + 8
    q = q.to(torch.uint8).flatten(-2)
    return types.SimpleNamespace(codes=q[:, 0::2] | q[:, 1::2] << 4, scales=scales, zeros=zeros)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(torch.bfloat16)

    def channels(x):  # a few channels are several times larger than the rest
        gain = 1 + 5 * (torch.rand(x.shape[-1], generator=gen, device="cuda") < 0.05)
        return (x.float() * gain).to(torch.bfloat16)

    def lens(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    s = types.SimpleNamespace(case=case)
    op = case["op"]
    if op == "norm":
        b, n, d = case["batch"], case["seq"], case["dim"]
        s.h, s.x = channels(randn(b, n, d, scale=2.0)), channels(randn(b, n, d))
        s.gate = s.scale = s.shift = None
        if case["modulated"]:
            s.gate, s.scale, s.shift = (randn(b, 1, d, scale=0.5) for _ in range(3))

        def norm(kind):
            if kind == "rms":
                return types.SimpleNamespace(weight=(1 + 0.2 * randn(d)).to(torch.bfloat16), bias=None, eps=EPS)
            return types.SimpleNamespace(normalized_shape=(d,), elementwise_affine=False, eps=EPS) if kind == "layer" else None
        s.post, s.norm, s.alpha = norm(case["post"]), norm(case["norm"]), 0.75
    elif op == "four":
        s.x = channels(randn(case["rows"], case["k"]))
        s.weights = [_four_bits(channels(randn(case["n"], case["k"], scale=case["k"] ** -0.5)), case)
                     for _ in range(2 if case["swiglu"] else 1)]
        s.bias = randn(case["n"]) if case["bias"] and not case["swiglu"] else None
        if own:
            fourbit = _kernels()[2]
            s.packed = [fourbit.pack_weight(w.codes, w.scales, zeros=w.zeros) for w in s.weights]
    else:
        b, t, kv, c = case["batch"], case["prefix"], case["kv_heads"], case["capacity"]
        s.q = randn(b, case["seq"], case["heads"], HEAD)
        s.prefix = [*_quantized(channels(randn(case["prefixes"], t, kv, HEAD))), *_quantized(randn(case["prefixes"], t, kv, HEAD))]
        s.cache = [*_quantized(channels(randn(b, c, kv, HEAD))), *_quantized(randn(b, c, kv, HEAD))]
        s.lengths, s.prefix_lengths, s.share = lens(_lengths(case)), lens(_prefix_lengths(case)), lens(_share(case))
        s.tree = _tree(b, case["seq"], seed).cuda() if case["tree"] else None
    return s


# -------------------------------------------------------------------- runs --

def run(s):
    if own:
        return _own(s)
    return {"norm": _norm, "four": _four, "share": _shared}[s.case["op"]](s)


def _kernels():
    """The framework's modules, imported once."""
    if not _modules:
        if PKG not in sys.path:
            sys.path.insert(0, PKG)
        from qwen_image_accel.kernels import attention, elementwise, fourbit, kv_cache
        _modules.extend((attention, elementwise, fourbit, kv_cache))
    return _modules


_modules = []


def _own(s):
    attention, elementwise, fourbit, kv_cache = _kernels()
    op = s.case["op"]
    if op == "norm":
        return elementwise.residual_norm(s.h, s.x, s.norm, gate=s.gate, residual_scale=s.alpha, post=s.post, scale=s.scale,
                                         shift=s.shift, add_one=True)
    if op == "four":
        if s.case["swiglu"]:
            return fourbit.swiglu(s.x, *s.packed)
        return fourbit.matmul(s.x, s.packed[0], bias=s.bias)
    share = None if s.case["prefixes"] == 1 else s.share
    return attention.attention_shared(s.q, kv_cache.QuantizedCache(*s.prefix), kv_cache.QuantizedCache(*s.cache), s.lengths,
                                      share=share, prefix_lengths=s.prefix_lengths, tree=s.tree)


def _normed(x, norm):
    if hasattr(norm, "normalized_shape"):
        x = x - x.mean(-1, keepdim=True)
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + norm.eps)
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + norm.eps) * norm.weight.float()


def _norm(s):
    u = s.x.float()
    if s.post is not None:
        u = _normed(u, s.post)
    if s.gate is not None:
        u = u * s.gate.float()
    h = s.h.float() + s.alpha * u
    z = _normed(h, s.norm)
    if s.scale is not None:
        z = z * (1 + s.scale.float()) + s.shift.float()
    return h.to(torch.bfloat16), z.to(torch.bfloat16)


def _weight(w, case):
    """The float32 weight (N, K) that the codes stand for."""
    q = torch.stack([w.codes & 15, w.codes >> 4], dim=-1).flatten(-2)
    if case["kind"] == "mxfp4":
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=q.device)
        return (table[q.int()].unflatten(-1, (-1, 32)) * torch.exp2(w.scales.float() - 127).unsqueeze(-1)).flatten(-2)
    zeros = 8.0 if w.zeros is None else w.zeros.float().unsqueeze(-1)
    return ((q.float().unflatten(-1, (-1, case["group"])) - zeros) * w.scales.float().unsqueeze(-1)).flatten(-2)


def _four(s):
    y = [torch.matmul(s.x.float(), _weight(w, s.case).t()) for w in s.weights]
    if s.case["swiglu"]:
        return (y[0] / (1 + torch.exp(-y[0])) * y[1]).to(torch.bfloat16)
    return (y[0] if s.bias is None else y[0] + s.bias.float()).to(torch.bfloat16)


def _visible(s, b, n, t):
    """(B, 1, 1, S, C): which of its own keys a query sees."""
    at = torch.arange(t, device="cuda")
    seen = (at < s.lengths[:, None])[:, None].expand(b, n, t)
    if s.tree is not None:
        j = at - (s.lengths[:, None] - n)                                       # (B, C): place among the drafted tokens
        own_mask = s.tree.gather(2, j.clamp(0, n - 1)[:, None].expand(b, n, t))
        seen = seen & (own_mask | (j < 0)[:, None])
    return seen[:, None, None]


def _shared(s):
    b, n, h, d = s.q.shape
    kv = s.case["kv_heads"]
    q = s.q.float().unflatten(2, (kv, -1)).permute(0, 2, 3, 1, 4) * d ** -0.5    # (B, KV, G, S, D)
    k, v = (_values(c, e).transpose(1, 2).contiguous() for c, e in (s.cache[:2], s.cache[2:]))      # (B, KV, C, D)
    w = torch.matmul(q.flatten(2, 3), k.transpose(2, 3)).unflatten(2, (-1, n))
    w = w.masked_fill(~_visible(s, b, n, k.shape[2]), -math.inf)
    top = w.amax(-1, keepdim=True)                                              # (B, KV, G, S, 1)
    parts = []                                                                  # per prefix: its requests, scores, values
    for i, length in enumerate(_prefix_lengths(s.case)):
        mine = [j for j, p in enumerate(_share(s.case)) if p == i]
        if not mine:
            continue
        pk, pv = (_values(c[i, :length], e[i, :length]).transpose(0, 1).contiguous()
                  for c, e in (s.prefix[:2], s.prefix[2:]))                     # (KV, T, D)
        rows = q[mine].permute(1, 0, 2, 3, 4).flatten(1, 3)                     # (KV, rows, D)
        scores = torch.matmul(rows, pk.transpose(1, 2))
        best = scores.amax(-1).unflatten(1, (len(mine), -1, n)).transpose(0, 1).unsqueeze(-1)
        top[mine] = torch.maximum(top[mine], best)
        parts.append((mine, scores, pv))
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(w - top)
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.flatten(2, 3), v).unflatten(2, (-1, n))
    for mine, scores, pv in parts:
        e = torch.exp(scores - top[mine].transpose(0, 1).flatten(1, 4).unsqueeze(-1))
        total[mine] += e.sum(-1).unflatten(1, (len(mine), -1, n)).transpose(0, 1).unsqueeze(-1)
        o[mine] += torch.matmul(e, pv).unflatten(1, (len(mine), -1, n)).transpose(0, 1)
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, h, d).to(torch.bfloat16)


def work(case):
    op = case["op"]
    if op == "norm":
        rows, d = case["batch"] * case["seq"], case["dim"]
        vectors = 2 * d * ((3 * case["batch"] if case["modulated"] else 0) + (case["post"] == "rms") + (case["norm"] == "rms"))
        return {"bytes": 8 * rows * d + vectors, "flops": 16 * rows * d}
    if op == "four":
        m, n, k, times = case["rows"], case["n"], case["k"], 2 if case["swiglu"] else 1
        per_group = (1 if case["kind"] == "mxfp4" else 2) + (1 if case["zeros"] else 0)
        bias = 2 * n if case["bias"] and not case["swiglu"] else 0
        return {"bytes": times * (n * k // 2 + n * (k // case["group"]) * per_group) + 2 * m * (k + n) + bias,
                "flops": 2 * times * m * n * k}
    share, lengths = _share(case), _prefix_lengths(case)
    prefix = sum(n for i, n in enumerate(lengths) if i in share)
    own_keys = sum(_lengths(case))
    row_keys = sum(lengths[p] for p in share if p >= 0) + own_keys
    return {"bytes": (prefix + own_keys) * case["kv_heads"] * 2 * (HEAD + HEAD // 32)
                     + 4 * case["batch"] * case["seq"] * case["heads"] * HEAD,
            "flops": 4 * case["seq"] * case["heads"] * HEAD * row_keys}


# ------------------------------------------------- the definitions in 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "four": _exact_four, "share": _exact_shared}[case["op"]](s)


def _exact_norm(s):
    def normalised(y, kind, norm):
        if kind == "none":
            return y
        if kind == "layer":
            var, mean = torch.var_mean(y, dim=-1, correction=0, keepdim=True)
            return (y - mean) / torch.sqrt(var + norm.eps)
        return y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + norm.eps) * norm.weight.double()
    u = normalised(s.x.double(), s.case["post"], s.post)
    if s.case["modulated"]:
        u = s.gate.double() * u
    h = torch.add(s.h.double(), u, alpha=s.alpha)
    z = normalised(h, s.case["norm"], s.norm)
    return h, (1.0 + s.scale.double()) * z + s.shift.double() if s.case["modulated"] else z


def _exact_four(s):
    def weight(w):
        n, k = w.codes.shape[0], 2 * w.codes.shape[1]
        q = torch.empty(n, k, dtype=torch.float64, device=w.codes.device)
        for half in (0, 1):
            c = (w.codes.int() >> (4 * half)) % 16
            if s.case["kind"] == "mxfp4":  # sign, two exponent bits, one fraction bit; exponent 0 without the leading one
                e, f = (c >> 1) % 4, (c % 2).double()
                mag = torch.where(e == 0, f / 2, (1 + f / 2) * torch.exp2((e - 1).double()))
                q[:, half::2] = torch.where(c >= 8, -mag, mag)
            else:
                q[:, half::2] = c.double()
        per = s.case["group"]
        if s.case["kind"] == "mxfp4":
            return q * torch.exp2(w.scales.double() - 127).repeat_interleave(per, 1)
        z = torch.full_like(w.scales, 8).double() if w.zeros is None else w.zeros.double()
        return (q - z.repeat_interleave(per, 1)) * w.scales.double().repeat_interleave(per, 1)
    x = s.x.double()
    y = x @ weight(s.weights[0]).T
    if s.case["swiglu"]:
        return y * torch.sigmoid(y) * (x @ weight(s.weights[1]).T)
    return y if s.bias is None else y + s.bias.double()


def _exact_shared(s):
    def stored(codes, exponents):
        return (codes.double().unflatten(-1, (-1, 32)) * torch.exp2(exponents.double() - 127)[..., None]).flatten(-2)
    b, n, h, d = s.q.shape
    kv, share, spans = s.case["kv_heads"], _share(s.case), _prefix_lengths(s.case)
    group, out = h // kv, torch.zeros(b, n, h, d, dtype=torch.float64, device="cuda")
    kc, ke, vc, ve = s.prefix
    oc, oe, wc, we = s.cache
    for j in range(kv):
        front = {p: (stored(kc[p, :spans[p], j], ke[p, :spans[p], j]), stored(vc[p, :spans[p], j], ve[p, :spans[p], j]))
                 for p in set(share) if p >= 0}
        for i in range(b):
            t = int(s.lengths[i])
            k, v = stored(oc[i, :t, j], oe[i, :t, j]), stored(wc[i, :t, j], we[i, :t, j])
            seen = torch.ones(n, t, dtype=torch.bool, device="cuda")
            if s.tree is not None:
                seen[:, t - n:] = s.tree[i]
            if share[i] >= 0:
                fk, fv = front[share[i]]
                k, v = torch.cat([fk, k]), torch.cat([fv, v])
                seen = torch.cat([torch.ones(n, len(fk), dtype=torch.bool, device="cuda"), seen], dim=1)
            q = s.q[i, :, j * group:(j + 1) * group].double().transpose(0, 1)       # (G, S, D)
            w = (q @ k.T) / math.sqrt(d)
            out[i, :, j * group:(j + 1) * group] = (torch.softmax(w.masked_fill(~seen, -math.inf), -1) @ v).transpose(0, 1)
    return out
