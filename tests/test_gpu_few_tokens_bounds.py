"""Attention over shared prefixes and 4-bit products against bounds that count the kernels' own roundings, on random values, on
values that cancel, and on keys that each stand out in some row."""
import random

import pytest
import torch

from qwen_image_accel.kernels import attention, fourbit, kv_cache
from tests import few_tokens_bounds as B
from tests.helpers import bf16_randn

pytestmark = pytest.mark.gpu

# (requests, tokens, heads, K/V heads, prefixes, prefix capacity, own capacity): up to 16, 32, 64 and more rows on a prefix, several
# prefixes found by every wave and (above 64 requests or 16 prefixes) by a launch of their own, pieces of one and of many blocks
SHAPES = [(1, 1, 1, 1, 1, 1, 1), (3, 1, 4, 1, 1, 64, 40), (16, 1, 4, 4, 1, 1101, 96), (17, 1, 8, 2, 1, 700, 70), (5, 7, 5, 5, 1, 65, 7), (8, 24, 2, 2, 1, 515, 40),
          (64, 1, 4, 1, 1, 2000, 20), (32, 2, 8, 4, 1, 3001, 100), (2, 64, 2, 1, 1, 190, 64), (1, 1, 8, 8, 1, 12000, 300), (40, 1, 16, 8, 1, 8000, 33),
          (9, 5, 4, 2, 4, 130, 40), (48, 1, 8, 2, 5, 900, 33), (70, 1, 2, 1, 3, 257, 6), (20, 1, 2, 2, 70, 65, 3), (64, 3, 8, 2, 15, 130, 10), (40, 1, 2, 2, 17, 90, 5)]


def say(*a):
    print("[case]", *a, flush=True)


def ints(values, dev):
    return torch.tensor(list(values), dtype=torch.int32, device=dev)


def cache_of(dev, k, v):
    cache = kv_cache.empty_cache(*k.shape[:3], 128, dev)
    if k.shape[1]:
        kv_cache.write_cache(cache, k.to(torch.bfloat16).to(dev), v.to(torch.bfloat16).to(dev))
    return cache


def plan(b, p, cp, c, seed):
    """(lengths, share, prefix lengths): uneven, some requests on no prefix where there are several."""
    r = random.Random(seed)
    share = [0] * b if p == 1 else [r.choice([-1] + list(range(p)) * 3) for _ in range(b)]
    return [max(0, c - i % (c + 1)) for i in range(b)], share, [max(1, cp - i * 7 % cp) for i in range(p)]


def run(dev, q, prefix, cache, lengths, share, plens, tree=None):
    names = None if len(plens) == 1 else ints(share, dev)
    return attention.attention_shared(q, prefix, cache, ints(lengths, dev), share=names, prefix_lengths=ints(plens, dev),
                                      tree=None if tree is None else tree.to(dev)).double().cpu()


def inside(got, want, bound, what=""):
    err = (got - want).abs()
    assert got.isfinite().all() and (err <= bound).all(), (what, float((err / bound).max()), (err > bound).nonzero()[:4].tolist())


@pytest.mark.parametrize("shape", SHAPES + [(1, 1, 8, 8, 1, 20000, 300)], ids=str)
def test_random_values(dev, shape):
    say("random", shape)
    b, s, h, hk, p, cp, c = shape
    g = torch.Generator().manual_seed(b + cp)
    q = bf16_randn(g, (b, s, h, 128)).to(dev)
    caches = [cache_of(dev, bf16_randn(g, (m, t, hk, 128)), bf16_randn(g, (m, t, hk, 128))) for m, t in ((p, cp), (b, c))]
    at = plan(b, p, cp, c, cp)
    o, e = B.attention_shared(q, *(kv_cache.read_cache(t) for t in caches), *at)
    inside(run(dev, q, *caches, *at), o, B.rounded(o, e))


@pytest.mark.parametrize("shape", [(2, 1, 4, 2, 1, 2, 2), (8, 1, 4, 1, 1, 6, 4), (20, 1, 4, 2, 1, 60, 2), (40, 1, 4, 1, 1, 130, 2), (3, 24, 4, 2, 1, 64, 30), (30, 1, 4, 2, 4, 40, 6)], ids=str)
def test_values_that_cancel(dev, shape):
    """Pairs of nearly equal keys with opposite values: what one bf16 rounding of p would leave stands out."""
    say("cancel", shape)
    b, s, h, hk, p, cp, c = shape
    g = torch.Generator().manual_seed(cp)
    q = bf16_randn(g, (b, s, h, 128)).to(dev)
    caches = []
    for m, t in ((p, cp), (b, c)):
        k, v = 0.3 * torch.randn(m, t, hk, 128, generator=g), 0.3 * torch.randn(m, t, hk, 128, generator=g)
        k[:, 1::2] = k[:, 0::2] + 0.05 * torch.randn(m, t // 2, hk, 128, generator=g)
        v[:, 1::2] = -v[:, 0::2]
        caches.append(cache_of(dev, k, v))
    at = ([c] * b, [i % p for i in range(b)], [cp] * p)
    o, e = B.attention_shared(q, *(kv_cache.read_cache(t) for t in caches), *at)
    inside(run(dev, q, *caches, *at), o, B.rounded(o, e))


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_every_key_counts_once(dev, shape, tree):
    """Queries of zeros: a row's output counts the keys it sees, place by place."""
    say("count", shape, tree)
    b, s, h, hk, p, cp, c = shape
    g = torch.Generator().manual_seed(cp + tree)
    values = [B.counted(g, (m, hk), t).transpose(1, 2).contiguous() for m, t in ((p, cp), (b, c))]
    prefix, cache = (cache_of(dev, torch.randn(v.shape, generator=g), v) for v in values)
    lengths, share, plens = plan(b, p, cp, c, cp)
    mask = (torch.rand(b, s, s, generator=g) < 0.6) if tree else None
    got = run(dev, torch.zeros(b, s, h, 128, dtype=torch.bfloat16, device=dev), prefix, cache, lengths, share, plens, mask)
    sums = {i: values[0][i, :plens[i]].double().sum(0) for i in set(share) if i >= 0}
    for i in range(b):
        pi, t, n = B.keys_of(i, lengths, share, plens, c, cp)
        seen = B.visible(s, t, n, None if mask is None else mask[i])[:, t:].double()
        own = torch.einsum("sn,nhd->shd", seen, values[1][i, :n].double())
        count = own + (sums[pi] if t else 0)
        total = (t + seen.sum(1)).clamp(min=1)[:, None, None]
        want = (count / total).repeat_interleave(h // hk, 1)
        inside(got[i], want, B.HALF * want + 8 * B.F32 * want, i)       # sums of ones are exact: a reciprocal, a product, the rounding


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rows_that_look_for_one_key(dev, shape):
    """Every row's query is some key, 16 times: its output is that key's value."""
    say("one key", shape)
    b, s, h, hk, p, cp, c = shape
    g = torch.Generator().manual_seed(cp)
    keys = [B.signs(g, (m, t, hk, 128)) for m, t in ((p, cp), (b, c))]
    prefix, cache = (cache_of(dev, k, bf16_randn(g, k.shape)) for k in keys)
    values = [kv_cache.read_cache(t)[1].double().cpu() for t in (prefix, cache)]
    lengths, share, plens = plan(b, p, cp, c, cp)
    rounds = max(1, min(6, max(len(B.edges(cp)), len(B.edges(c))) // max(1, b * s * h // p)))
    at = 0
    for _ in range(rounds):
        q, want, none = torch.zeros(b, s, h, 128), torch.zeros(b, s, h, 128, dtype=torch.float64), torch.zeros(b, s, h, dtype=torch.bool)
        for i in range(b):
            pi, t, n = B.keys_of(i, lengths, share, plens, c, cp)
            places = [(0, pi, k) for k in B.edges(t)] * 3 + [(1, i, k) for k in B.edges(n)]
            for j in range(s):
                for m in range(h):
                    if not places:
                        none[i, j, m] = True
                        continue
                    at += 1
                    where, seq, k = places[(at * 5 + i) % len(places)]
                    q[i, j, m] = 16 * keys[where][seq, k, m // (h // hk)]
                    want[i, j, m] = values[where][seq, k, m // (h // hk)]
        got = run(dev, q.to(torch.bfloat16).to(dev), prefix, cache, lengths, share, plens)
        # Another key's signs agree in d of 128 places more than not, d some 11 in deviation: it weighs e^(1.41 (d - 128)), less
        # than 2^-20 beside the row's own key up to d 118.
        inside(got, want, B.HALF * want.abs() + 2.0 ** -20, "one key")
        assert not got[none].any()


def test_keys_beyond_32_bits_of_a_prefix(dev):
    """The last of three prefixes of 2.1 GB of codes: rows that look for one of its first and last keys, zeros between."""
    say("far keys")
    p, cp, hk, near = 3, 262144 + 64, 64, 100
    codes = [torch.zeros(p, cp, hk, 128, dtype=torch.uint8, device=dev) for _ in range(2)]
    exponents = [torch.zeros(p, cp, hk, 4, dtype=torch.uint8, device=dev) for _ in range(2)]
    prefix = kv_cache.QuantizedCache(codes[0].view(torch.float8_e4m3fn), exponents[0], codes[1].view(torch.float8_e4m3fn), exponents[1])
    g = torch.Generator().manual_seed(1)
    keys = B.signs(g, (2, near, hk, 128))                                # the first keys, the last keys
    ends = cache_of(dev, keys, bf16_randn(g, keys.shape))
    for t, u in zip(prefix, ends):
        t[2, :near].view(torch.uint8).copy_(u[0].view(torch.uint8))
        t[2, cp - near:].view(torch.uint8).copy_(u[1].view(torch.uint8))
    values = kv_cache.read_cache(ends)[1].double().cpu()
    own = cache_of(dev, torch.zeros(6, 4, hk, 128), bf16_randn(g, (6, 4, hk, 128)))
    for b in (1, 6, 3):
        s = 64 if b == 3 else 8
        end, k = torch.randint(0, 2, (b, s, hk), generator=g), torch.randint(0, near, (b, s, hk), generator=g)
        head = torch.arange(hk).expand(b, s, hk)
        q = (16 * keys[end, k, head]).to(torch.bfloat16).to(dev)
        mine = kv_cache.QuantizedCache(*(t[:b] for t in own))
        got = attention.attention_shared(q, prefix, mine, ints([4] * b, dev), share=ints([2] * b, dev), prefix_lengths=ints([0, 0, cp], dev))
        want = values[end, k, head]
        inside(got.double().cpu(), want, B.HALF * want.abs() + 2.0 ** -20, b)


KINDS = [("int4", 32, True), ("int4", 64, True), ("int4", 128, True), ("int4", 64, False), ("mxfp4", 32, False)]


def random_weight(dev, g, n, k, kind, group, zeros):
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    if kind == "mxfp4":
        scales = torch.randint(112, 122, (n, k // 32), generator=g, dtype=torch.uint8)
    else:
        scales = (torch.rand(n, k // group, generator=g) * 0.02 - 0.001).to(torch.bfloat16)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    return tuple(None if t is None else t.to(dev) for t in (codes, scales, z))


@pytest.mark.parametrize("kind,group,zeros", KINDS)
@pytest.mark.parametrize("m,n,k", [(1, 16, 256), (3, 100, 4096), (4, 1001, 12288), (16, 48, 4096), (16, 6200, 1152), (33, 64, 2176), (65, 30, 256), (257, 96, 512),
                                   (24, 24610, 384), (70, 20000, 256), (1020, 4090, 384), (48, 12200, 640)])
def test_products_in_fp32(dev, m, n, k, kind, group, zeros):
    say("product", m, n, k, kind, group, zeros)
    g = torch.Generator().manual_seed(m + n)
    raw = random_weight(dev, g, n, k, kind, group, zeros)
    x = bf16_randn(g, (m, k)).to(dev)
    y, e = B.four_bit(x, *raw)
    got = fourbit.matmul(x, fourbit.pack_weight(raw[0], raw[1], zeros=raw[2]), dtype=torch.float32)
    inside(got.double().cpu(), y, B.rounded(y, e, torch.float32))


@pytest.mark.parametrize("m", [2, 16, 40, 300])
def test_the_ends_of_the_exponents(dev, m):
    """Weights around 2^-128 and, in codes that do not pass it, 2^127; scales of int4 below fp32's normal range."""
    say("ends", m)
    g = torch.Generator().manual_seed(m)
    n, k = 100, 384
    x = bf16_randn(g, (m, k))
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    low, high = (torch.randint(a, a + 3, (n, k // 32), generator=g, dtype=torch.uint8) for a in (0, 252))
    sub = (torch.rand(n, k // 64, generator=g) * 2.0 ** -127).to(torch.bfloat16)
    small = codes & 0xbb                                                 # 0, 0.5, 1, 1.5 and their negatives
    for c, scales, z, factor in ((codes, low, None, 2.0 ** 100), (small, high, None, 2.0 ** -40), (codes, sub, torch.randint(0, 16, sub.shape, generator=g, dtype=torch.uint8), 2.0 ** 90)):
        xs = (x.float() * factor).to(torch.bfloat16).to(dev)
        raw = [None if t is None else t.to(dev) for t in (c, scales, z)]
        y, e = B.four_bit(xs, *raw)
        got = fourbit.matmul(xs, fourbit.pack_weight(raw[0], raw[1], zeros=raw[2]), dtype=torch.float32)
        inside(got.double().cpu(), y, B.rounded(y, e, torch.float32), factor)


@pytest.mark.parametrize("group,zeros", [(32, True), (64, True), (128, False)])
@pytest.mark.parametrize("m", [2, 16, 40, 300])
def test_the_largest_values_of_x(dev, m, group, zeros):
    """Rows of bf16's largest numbers, of one sign or both: a group's sum of q - z times them is far beyond fp32, the result is not."""
    say("largest", m, group, zeros)
    g = torch.Generator().manual_seed(m + group)
    n, k = 100, 384
    codes, _, z = random_weight("cpu", g, n, k, "int4", group, zeros)
    scales = (torch.rand(n, k // group, generator=g) * 2.0 ** -20).to(torch.bfloat16)
    x = torch.full((m, k), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16)
    x[1::2] *= B.signs(g, x[1::2].shape).to(torch.bfloat16)
    x = x.to(dev)
    raw = [None if t is None else t.to(dev) for t in (codes, scales, z)]
    y, e = B.four_bit(x, *raw)
    w = fourbit.pack_weight(raw[0], raw[1], zeros=raw[2])
    for dtype in (torch.float32, torch.bfloat16):
        inside(fourbit.matmul(x, w, dtype=dtype).double().cpu(), y, B.rounded(y, e, dtype), dtype)
