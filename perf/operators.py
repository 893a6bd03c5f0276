"""Performance cases of the operators that serve many requests from one model: the K/V cache in MXFP8
(written, read back, packed in front of a step's keys), attention of a few tokens over that cache, and the
low-rank adapters of several requests beside a shared projection.

Sizes are those of the repository's configurations: 32 heads of 128 (hidden 4096) or 24, FFN 12288, images
of 1024 and 4096 tokens, prefixes of a few dozen text tokens up to another image's 4296, and generic ones
where those say nothing (shared K/V heads, long caches, adapter ranks).

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
        # One new token of each of 16 requests, every row with an adapter of its own: latency.
        {"name": "adapter_tokens", "op": "adapter", "batch": 16, "seq": 1, "k": 4096, "n": 4096, "rank": 16, "parts": 1,
         "adapters": 16, "rows": False},
        # An attention projection of two 512^2 requests, one adapter each.
        {"name": "adapter_512", "op": "adapter", "batch": 2, "seq": 1024, "k": 4096, "n": 4096, "rank": 32, "parts": 1,
         "adapters": 4, "rows": False},
        # The stacked Q/K/V projection of two 1024^2 requests: three rank slices, one read of the activation.
        {"name": "adapter_qkv_1024", "op": "adapter", "batch": 2, "seq": 4096, "k": 4096, "n": 12288, "rank": 16,
         "parts": 3, "adapters": 4, "rows": False},
        # The down projection over a packed batch of ragged requests, an index per row, some rows without an adapter.
        {"name": "adapter_packed_down", "op": "adapter", "batch": 1, "seq": 2381, "k": 12288, "n": 4096, "rank": 64,
         "parts": 1, "adapters": 6, "rows": True},
        # One new token of each of 16 requests written at its own position; a short cache read back.
        {"name": "cache_token", "op": "cache", "batch": 16, "seq": 1, "capacity": 128, "heads": 32, "dim": 128},
        # The prefix of an image-editing request (another image and the text) written once and staged back.
        {"name": "cache_edit", "op": "cache", "batch": 1, "seq": 4296, "capacity": 4296, "heads": 32, "dim": 128},
        # A 512^2 decode step, both guidance branches, a short text prefix in the cache.
        {"name": "pack_512", "op": "pack", "batch": 2, "seq": 1024, "prefix": 77, "heads": 32},
        # A 1024^2 editing step: the prefix is as long as the target.
        {"name": "pack_edit", "op": "pack", "batch": 1, "seq": 4096, "prefix": 4296, "heads": 32},
        # One token of one request over a short cache: latency.
        {"name": "attend_token", "op": "attend", "batch": 1, "seq": 1, "length": 1101, "heads": 32, "kv_heads": 32,
         "tree": False},
        # One token of each of 16 requests over caches of different lengths.
        {"name": "attend_batch", "op": "attend", "batch": 16, "seq": 1, "length": 8392, "heads": 32, "kv_heads": 32,
         "tree": False},
        # 24 drafted tokens of each of 4 requests, a tree per request.
        {"name": "attend_tree", "op": "attend", "batch": 4, "seq": 24, "length": 8392, "heads": 32, "kv_heads": 32,
         "tree": True},
        # Two long contexts, 4 query heads to a K/V head.
        {"name": "attend_long_shared", "op": "attend", "batch": 2, "seq": 1, "length": 131072, "heads": 32, "kv_heads": 8,
         "tree": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("adapter", "adapter", "cache", "pack", "attend", "attend"))
    if op == "adapter":
        rows = rng.random() < 0.4
        total = _log(rng, 1, 6144)
        batch = 1 if rows else rng.randint(1, min(total, 64))
        return {"op": op, "batch": batch, "seq": max(1, total // batch), "k": 8 * _log(rng, 64, 1536),
                "n": 96 * _log(rng, 8, 128), "rank": 8 * rng.choice((1, 1, 2, 2, 3, 4, 5, 8, 16)), "parts": rng.choice((1, 1, 2, 3)),
                "adapters": rng.randint(1, 24), "rows": rows}
    if op == "cache":
        batch, seq = _log(rng, 1, 16), _log(rng, 1, 4096)
        seq = max(1, min(seq, 4096 // batch))
        return {"op": op, "batch": batch, "seq": seq, "capacity": min(seq + _log(rng, 1, 256), max(seq, 4296 // batch)),
                "heads": rng.choice((8, 20, 24, 32)), "dim": rng.choice((64, 128, 128))}
    if op == "pack":
        return {"op": op, "batch": rng.randint(1, 2), "seq": _log(rng, 16, 2048), "prefix": _log(rng, 1, 2048),
                "heads": rng.choice((16, 20, 24, 32))}
    kv = rng.choice((4, 8, 16, 32))
    heads = kv * rng.choice((1, 1, 2, 4)) if kv < 16 else kv
    batch = _log(rng, 1, 32)
    seq = rng.choice((1, 1, 2, 5, 16, 33, 64))
    most = max(seq, min(65536, 8192 * 16 * 32 // (batch * kv * (1 + seq * heads // kv // 32))))
    return {"op": op, "batch": batch, "seq": seq, "length": _log(rng, seq, most), "heads": heads, "kv_heads": kv,
            "tree": seq > 1 and rng.random() < 0.7}


# ------------------------------------------------------------------ inputs --

def _lengths(case):
    """Valid keys of each sequence: the longest first, down to about half of it, never below the drafted tokens."""
    b, t = case["batch"], case["length"]
    return [max(case["seq"], t - t * i // (2 * b)) for i in range(b)]


def _places(case):
    """(first position, number of rows) that each sequence writes: anywhere that fits, the last sequences fewer rows."""
    out = []
    for i in range(case["batch"]):
        n = max(1, case["seq"] - case["seq"] * i // (2 * case["batch"]))
        out.append(((7 * i) % (case["capacity"] - case["seq"] + 1), n))
    return out


def _index(case):
    """The adapter of each row group: every fifth has none; with "rows", runs of ragged lengths over the rows."""
    r = random.Random(case["batch"] * 1009 + case["seq"])
    if not case["rows"]:
        return [-1 if i % 5 == 4 else i % case["adapters"] for i in range(case["batch"])]
    out = []
    while len(out) < case["seq"]:
        out += [r.choice([-1] + list(range(case["adapters"])))] * r.randint(1, max(1, case["seq"] // 6))
    return out[:case["seq"]]


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


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(torch.bfloat16)

    def channels(x):  # a few channels of a head are several times larger than the rest
        gain = 1 + 5 * (torch.rand(x.shape[-1], generator=gen, device="cuda") < 0.05)
        return (x.float() * gain).to(torch.bfloat16)

    s = types.SimpleNamespace(case=case)
    b, op = case["batch"], case["op"]
    if op == "adapter":
        m, k, n, r, a = b * case["seq"], case["k"], case["n"], case["rank"], case["adapters"]
        s.x = randn(m, k) if case["rows"] else randn(b, case["seq"], k)
        s.base = randn(*s.x.shape[:-1], n)
        s.down = randn(a, case["parts"] * r, k, scale=k ** -0.5)
        s.up = randn(a, n, r, scale=0.5 * r ** -0.5)
        s.scale = 0.25 + torch.rand(a, generator=gen, device="cuda")
        s.index = torch.tensor(_index(case), dtype=torch.int32, device="cuda")
    elif op == "cache":
        h, d, c = case["heads"], case["dim"], case["capacity"]
        s.k, s.v = channels(randn(b, case["seq"], h, d)), randn(b, case["seq"], h, d)
        old = channels(randn(b, c, h, d, scale=2.0))
        (s.ck, s.ek), (s.cv, s.ev) = _quantized(old), _quantized(old.flip(1))
        places = _places(case)
        s.start = torch.tensor([p for p, _ in places], dtype=torch.int32, device="cuda")
        s.count = torch.tensor([n for _, n in places], dtype=torch.int32, device="cuda")
    elif op == "pack":
        h, t = case["heads"], case["seq"]
        qkv = randn(b, t, 3, h, HEAD)                         # one fused projection's output
        s.q, s.k, s.v = qkv.unbind(2)
        (s.ck, s.ek), (s.cv, s.ev) = (_quantized(channels(randn(b, case["prefix"], h, HEAD))) for _ in range(2))
        s.norm_q, s.norm_k = (types.SimpleNamespace(weight=(1 + 0.2 * randn(HEAD)).to(torch.bfloat16), eps=EPS, bias=None)
                              for _ in range(2))
        angle = torch.outer(torch.arange(t).double(), 10000.0 ** (-torch.arange(0, HEAD, 2).double() / HEAD))
        s.freqs = torch.polar(torch.ones_like(angle), angle).to(torch.complex64).cuda()
    else:
        t, kv = case["length"], case["kv_heads"]
        s.q = randn(b, case["seq"], case["heads"], HEAD)
        (s.ck, s.ek), (s.cv, s.ev) = _quantized(channels(randn(b, t, kv, HEAD))), _quantized(randn(b, t, kv, HEAD))
        s.lengths = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        s.tree = _tree(b, case["seq"], seed).cuda() if case["tree"] else None
    return s


# -------------------------------------------------------------------- runs --

def run(s):
    if own:
        return _own(s)
    return {"adapter": _adapter, "cache": _cache, "pack": _pack, "attend": _attend}[s.case["op"]](s)


def _kernels():
    """The framework's modules, imported once."""
    if not _modules:
        if PKG not in sys.path:
            sys.path.insert(0, PKG)
        from qwen_image_accel.kernels import adapters, attention, kv_cache
        _modules.extend((adapters, attention, kv_cache))
    return _modules


_modules = []


def _own(s):
    adapters, attention, kv_cache = _kernels()
    op = s.case["op"]
    if op == "adapter":
        return adapters.low_rank(s.x, s.down, s.up, s.index, scale=s.scale, base=s.base, parts=s.case["parts"])
    cache = kv_cache.QuantizedCache(s.ck, s.ek, s.cv, s.ev)
    if op == "cache":
        kv_cache.write_cache(cache, s.k, s.v, start=s.start, count=s.count)
        return kv_cache.read_cache(cache)
    if op == "pack":
        return attention.prepare_attention_inputs_quantized(s.q, s.k, s.v, s.norm_q, s.norm_k, s.freqs, cache)
    return attention.attention_cached(s.q, cache, s.lengths, tree=s.tree)


def _adapter(s):
    parts, r = s.case["parts"], s.case["rank"]
    index = s.index.long()
    live, a = index >= 0, index.clamp(min=0)
    x = s.x.float() if s.x.dim() == 3 else s.x.float().unsqueeze(1)            # (groups, rows, K)
    if s.x.dim() == 3:
        h = torch.matmul(x, s.down.float()[a].transpose(1, 2))                 # (groups, rows, parts r)
        h = h.unflatten(-1, (parts, r)).transpose(1, 2)                        # (groups, parts, rows, r)
        up = s.up.float()[a].unflatten(1, (parts, -1)).transpose(2, 3)         # (groups, parts, r, N / parts)
        delta = torch.matmul(h, up).transpose(1, 2).flatten(2)
    else:  # an index per row: every adapter over all rows, then each row's own
        h = torch.matmul(s.x.float(), s.down.float().flatten(0, 1).t()).unflatten(1, (-1, parts, r))
        mine = torch.nn.functional.one_hot(a, s.down.shape[0]).float()[:, :, None, None] * h        # (rows, A, parts, r)
        up = s.up.float().unflatten(1, (parts, -1))                            # (A, parts, N / parts, r)
        up = up.permute(1, 0, 3, 2).flatten(1, 2)                              # (parts, A r, N / parts)
        delta = torch.matmul(mine.permute(2, 0, 1, 3).flatten(2), up).permute(1, 0, 2).flatten(1).unsqueeze(1)
    delta = torch.where(live[:, None, None], s.scale[a][:, None, None] * delta, torch.zeros((), device=delta.device))
    return (s.base.float() + delta.view(s.base.shape)).to(torch.bfloat16)


def _cache(s):
    b, n = s.k.shape[:2]
    row = torch.arange(n, device="cuda")
    take = (row < s.count[:, None]).nonzero(as_tuple=True)
    at = take[0], (s.start[:, None] + row)[take]
    for x, codes, exponents in ((s.k, s.ck, s.ek), (s.v, s.cv, s.ev)):
        c, e = _quantized(x[take])
        codes.view(torch.uint8)[at] = c.view(torch.uint8)
        exponents[at] = e
    return _values(s.ck, s.ek).to(torch.bfloat16), _values(s.cv, s.ev).to(torch.bfloat16)


def _rotated(x, norm, freqs):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + norm.eps) * norm.weight.float()
    x0, x1 = x.unflatten(-1, (-1, 2)).unbind(-1)
    c, s = freqs.real[:, None], freqs.imag[:, None]
    return torch.stack([x0 * c - x1 * s, x0 * s + x1 * c], dim=-1).flatten(-2).to(torch.bfloat16)


def _pack(s):
    return (_rotated(s.q, s.norm_q, s.freqs),
            torch.cat([_values(s.ck, s.ek).to(torch.bfloat16), _rotated(s.k, s.norm_k, s.freqs)], dim=1),
            torch.cat([_values(s.cv, s.ev).to(torch.bfloat16), s.v], dim=1))


def _visible(s, b, n, t):
    """(B, 1, 1, S, T): which keys a query sees."""
    at = torch.arange(t, device="cuda")
    seen = (at < s.lengths[:, None])[:, None].expand(b, n, t)
    if s.tree is not None:
        j = at - (s.lengths[:, None] - n)                                       # (B, T): place among the drafted tokens
        own_mask = s.tree.gather(2, j.clamp(0, n - 1)[:, None].expand(b, n, t))
        seen = seen & (own_mask | (j < 0)[:, None])
    return seen[:, None, None]


def _attend(s):
    b, n, h, d = s.q.shape
    t, kv = s.ck.shape[1:3]
    q = s.q.float().unflatten(2, (kv, -1)).permute(0, 2, 3, 1, 4)               # (B, KV, G, S, D)
    k, v = (_values(c, e).transpose(1, 2).contiguous() for c, e in ((s.ck, s.ek), (s.cv, s.ev)))      # (B, KV, T, D)
    scores = torch.matmul(q.flatten(2, 3), k.transpose(2, 3)).unflatten(2, (-1, n)) * d ** -0.5
    scores = scores.masked_fill(~_visible(s, b, n, t), -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (-1, n)) / torch.where(total == 0, torch.ones_like(total), total)
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, h, d).to(torch.bfloat16)


def work(case):
    b, n, op = case["batch"], case["seq"], case["op"]
    if op == "adapter":
        m, r = b * n, case["parts"] * case["rank"]
        index = _index(case)
        used = len({a for a in index if a >= 0})
        live = sum(a >= 0 for a in index) * (1 if case["rows"] else n)
        return {"bytes": 2 * (live * case["k"] + 2 * m * case["n"] + used * (r * case["k"] + case["n"] * case["rank"])) + 4 * len(index),
                "flops": 2 * live * (case["k"] * r + case["n"] * case["rank"])}
    if op == "cache":
        width = case["heads"] * case["dim"]
        rows = sum(c for _, c in _places(case))
        coded = 33 * width // 32
        return {"bytes": 2 * (rows * (2 * width + coded) + b * case["capacity"] * (coded + 2 * width)), "flops": 0}
    if op == "pack":
        width = case["heads"] * HEAD
        return {"bytes": b * (n * width * 12 + 2 * case["prefix"] * (33 * width // 32 + 2 * width)) + n * HEAD * 4,
                "flops": 20 * b * n * width}
    keys = sum(_lengths(case))
    return {"bytes": keys * case["kv_heads"] * 2 * (HEAD + HEAD // 32) + 4 * b * n * case["heads"] * HEAD,
            "flops": 4 * n * case["heads"] * HEAD * keys}


# ------------------------------------------------- the definitions in 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    return {"adapter": _exact_adapter, "cache": _exact_cache, "pack": _exact_pack, "attend": _exact_attend}[case["op"]](s)


def _exact_adapter(s):
    parts, r = s.case["parts"], s.case["rank"]
    x = s.x.double().reshape(-1, s.case["k"])
    y = s.base.double().reshape(-1, s.case["n"]).clone()
    rows_of = torch.repeat_interleave(s.index.long(), 1 if s.case["rows"] else s.case["seq"])
    width = s.case["n"] // parts
    for a in range(s.case["adapters"]):
        rows = (rows_of == a).nonzero()[:, 0]
        for j in range(parts):
            low = x[rows] @ s.down[a, j * r:(j + 1) * r].double().T
            y[rows, j * width:(j + 1) * width] += float(s.scale[a]) * (low @ s.up[a, j * width:(j + 1) * width].double().T)
    return y.view(s.base.shape)


def _exact_block_values(x):
    """What x (..., D) stands for once held in 8 bits: per 32 values a power of two, per value 4 significand bits, ties to even."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    unit = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(top.clamp(min=1e-300) / 448)).clamp(-127, 127)), torch.ones_like(top))
    y = g / unit
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))).clamp(-6, 8) - 3)
    return (torch.round(y / step) * step * unit).flatten(-2)


def _exact_stored(codes, exponents):
    return (codes.double().unflatten(-1, (-1, 32)) * torch.exp2(exponents.double() - 127)[..., None]).flatten(-2)


def _exact_cache(s):
    k, v = _exact_stored(s.ck, s.ek), _exact_stored(s.cv, s.ev)
    for i, (first, n) in enumerate(_places(s.case)):
        k[i, first:first + n] = _exact_block_values(s.k[i, :n])
        v[i, first:first + n] = _exact_block_values(s.v[i, :n])
    return k, v


def _exact_pack(s):
    def turned(x, norm):
        x = x.double()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + norm.eps) * norm.weight.double()
        z = torch.complex(x[..., 0::2], x[..., 1::2]) * s.freqs.to(torch.complex128)[None, :, None]
        return torch.view_as_real(z).flatten(-2)
    return (turned(s.q, s.norm_q), torch.cat([_exact_stored(s.ck, s.ek), turned(s.k, s.norm_k)], 1),
            torch.cat([_exact_stored(s.cv, s.ev), s.v.double()], 1))


def _exact_attend(s):
    b, n, h, d = s.q.shape
    group = h // s.ck.shape[2]
    out = torch.zeros(b, n, h, d, dtype=torch.float64, device="cuda")
    for i in range(b):
        t = int(s.lengths[i])
        k, v = _exact_stored(s.ck[i, :t], s.ek[i, :t]), _exact_stored(s.cv[i, :t], s.ev[i, :t])
        seen = torch.ones(n, t, dtype=torch.bool, device="cuda")
        if s.tree is not None:
            seen[:, t - n:] = s.tree[i]
        for j in range(h):
            w = (s.q[i, :, j].double() @ k[:, j // group].T) / math.sqrt(d)
            out[i, :, j] = torch.softmax(w.masked_fill(~seen, -math.inf), -1) @ v[:, j // group]
    return out
