"""Attention of many requests over shared prefixes against float64."""
import random

import pytest
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import attention, kv_cache
from tests import few_tokens_ref as R
from tests.helpers import bf16_randn

pytestmark = pytest.mark.gpu


def say(*a):
    print("[case]", *a, flush=True)


def filled(dev, g, b, c, hk, kscale=1.0):
    cache = kv_cache.empty_cache(b, c, hk, 128, dev)
    kv_cache.write_cache(cache, bf16_randn(g, (b, c, hk, 128), kscale).to(dev), bf16_randn(g, (b, c, hk, 128)).to(dev))
    return cache


def make(dev, b, s, h, hk, p, cp, c, seed=0, kscale=1.0):
    g = torch.Generator().manual_seed(seed)
    return bf16_randn(g, (b, s, h, 128)).to(dev), filled(dev, g, p, cp, hk, kscale), filled(dev, g, b, c, hk, kscale)


def ints(values, dev):
    return torch.tensor(list(values), dtype=torch.int32, device=dev)


def check(out, q, prefix, cache, lengths, share, plens, tree=None, scale=None):
    want, bound = R.attention_shared(q, kv_cache.read_cache(prefix), kv_cache.read_cache(cache), lengths, share, plens, tree, scale)
    err = (out.double().cpu() - want).abs()
    assert out.isfinite().all() and (err <= bound).all(), float((err / bound.clamp(min=1e-30)).max())


def random_tree(b, s, seed):
    g = torch.Generator().manual_seed(seed)
    m = torch.zeros(b, s, s, dtype=torch.bool)
    for i in range(b):
        for j in range(s):
            if j:
                m[i, j] = m[i, int(torch.randint(0, j, (1,), generator=g))]
            m[i, j, j] = True
    return m


@pytest.mark.parametrize("b,s,h,hk,cp,c", [
    (1, 1, 1, 1, 1, 1), (4, 1, 2, 2, 33, 5), (3, 1, 4, 1, 64, 40), (2, 3, 6, 2, 129, 33), (16, 1, 4, 4, 1101, 96), (17, 1, 8, 2, 700, 70),
    (5, 7, 5, 5, 65, 7), (33, 1, 2, 2, 300, 31), (2, 64, 2, 1, 190, 64), (40, 2, 3, 3, 96, 3), (8, 24, 2, 2, 515, 40),
    (64, 1, 4, 1, 2000, 20), (3, 33, 8, 2, 97, 64), (130, 1, 2, 2, 257, 9), (1, 1, 8, 8, 20000, 300)])
def test_one_prefix(dev, b, s, h, hk, cp, c):
    say("one prefix", b, s, h, hk, cp, c)
    q, prefix, cache = make(dev, b, s, h, hk, 1, cp, c, seed=b + cp)
    lengths = [max(0, c - i) for i in range(b)]
    out = attention.attention_shared(q, prefix, cache, ints(lengths, dev))
    check(out, q, prefix, cache, lengths, [0] * b, [cp])
    short = [cp // 2 + 1]
    out = attention.attention_shared(q, prefix, cache, ints(lengths, dev), prefix_lengths=ints(short, dev), scale=0.2)
    check(out, q, prefix, cache, lengths, [0] * b, short, scale=0.2)


@pytest.mark.parametrize("b,s,h,hk,p,cp,c", [
    (1, 1, 1, 1, 3, 40, 4), (6, 1, 2, 2, 2, 100, 8), (9, 5, 4, 2, 4, 130, 40), (48, 1, 8, 2, 5, 900, 33), (70, 1, 2, 1, 3, 257, 6),
    (20, 1, 2, 2, 70, 65, 3), (5, 33, 4, 4, 2, 300, 60), (150, 1, 1, 1, 6, 64, 2), (30, 3, 4, 4, 1, 333, 9),
    (64, 1, 4, 2, 16, 200, 9), (64, 3, 8, 2, 15, 130, 10), (65, 1, 2, 2, 16, 100, 5), (40, 1, 2, 2, 17, 90, 5), (40, 64, 4, 1, 2, 70, 64)])
def test_several_prefixes(dev, b, s, h, hk, p, cp, c):
    """Prefixes of different lengths, some of them empty or of no request, and requests without a prefix."""
    say("prefixes", b, s, h, hk, p, cp, c)
    r = random.Random(b * p)
    q, prefix, cache = make(dev, b, s, h, hk, p, cp, c, seed=b + p)
    share = [r.choice([-1, p, 1 << 30] + list(range(p)) * 3) for _ in range(b)]
    plens = [r.choice((0, -3, cp + 7, cp, cp // 2, cp // 3 + 1)) for _ in range(p)]
    lengths = [r.randint(0, c) for _ in range(b)]
    out = attention.attention_shared(q, prefix, cache, ints(lengths, dev), share=ints(share, dev), prefix_lengths=ints(plens, dev))
    check(out, q, prefix, cache, lengths, share, plens)


@pytest.mark.parametrize("b,s,h,hk,p,cp,c,shared", [
    (2, 2, 1, 1, 1, 40, 2, False), (3, 5, 2, 2, 2, 60, 12, False), (8, 24, 4, 4, 1, 500, 64, False), (2, 64, 2, 1, 1, 150, 100, True),
    (4, 33, 8, 2, 2, 97, 40, False), (2, 7, 4, 2, 1, 40, 20, True)])
def test_tree(dev, b, s, h, hk, p, cp, c, shared):
    """Trees over the last own keys, also where a request has fewer keys than the tree."""
    say("tree", b, s, h, hk, p, cp, c, shared)
    q, prefix, cache = make(dev, b, s, h, hk, p, cp, c, seed=s + c)
    tree = random_tree(b, s, s)
    tree = tree[0].contiguous() if shared else tree
    share = [i % (p + 1) - (p > 1) for i in range(b)] if p > 1 else [0] * b
    lengths = [c, max(0, s - 2)] + [s] * (b - 2)
    out = attention.attention_shared(q, prefix, cache, ints(lengths, dev), share=ints(share, dev), tree=tree.to(dev))
    check(out, q, prefix, cache, lengths, share, [cp] * p, tree)


def test_rows_that_see_nothing_are_zeros(dev):
    say("nothing")
    q, prefix, cache = make(dev, 5, 3, 4, 2, 2, 70, 9)
    tree = torch.zeros(5, 3, 3, dtype=torch.bool)
    tree[4, 1, 2] = True
    share, lengths, plens = [-1, 0, 1, -1, -1], [0, 0, 9, 3, 3], [0, 70]
    out = attention.attention_shared(q, prefix, cache, ints(lengths, dev), share=ints(share, dev), prefix_lengths=ints(plens, dev), tree=tree.to(dev))
    check(out, q, prefix, cache, lengths, share, plens, tree)
    assert not out[0].any() and not out[1].any() and not out[3].any() and out[2].any() and out[4, 1].any() and not out[4, 0].any()


def test_no_own_keys(dev):
    """An own cache of no positions: the prefix alone."""
    say("no own cache")
    q, prefix, _ = make(dev, 6, 2, 4, 2, 1, 200, 1)
    cache = kv_cache.empty_cache(6, 0, 2, 128, dev)
    out = attention.attention_shared(q, prefix, cache, ints([0] * 6, dev))
    want, bound = R.attention_shared(q, kv_cache.read_cache(prefix), [torch.zeros(6, 0, 2, 128)] * 2, [0] * 6, [0] * 6, [200])
    assert ((out.double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("b", [3, 14, 20, 70])
@pytest.mark.parametrize("falling", [False, True])
def test_scores_that_rise_or_fall_along_the_keys(dev, b, falling):
    """The row's maximum moves with every block of keys, by less and by more than what the sums leave room for."""
    say("rising", b, falling)
    h, hk, cp, c = 6, 2, 700, 40
    q, prefix, cache = make(dev, b, 1, h, hk, 1, cp, c, seed=b)
    g = torch.Generator().manual_seed(b + 1)
    along = bf16_randn(g, (1, 1, 1, 128)).float()
    steps = torch.linspace(-3, 3, cp)[None, :, None, None]
    k = (along * (steps.flip(1) if falling else steps)).expand(1, cp, hk, 128).to(torch.bfloat16).contiguous().to(dev)
    kv_cache.write_cache(prefix, k, bf16_randn(g, (1, cp, hk, 128)).to(dev))
    q = (along * torch.linspace(0.1, 3, b * h).view(b, 1, h, 1)).to(torch.bfloat16).to(dev)
    out = attention.attention_shared(q, prefix, cache, ints([c] * b, dev))
    check(out, q, prefix, cache, [c] * b, [0] * b, [cp])


@pytest.mark.parametrize("b", [2, 6, 14, 32])
def test_a_row_has_its_bits_whatever_the_others_hold(dev, b):
    """Other requests' large scores and NaN, over pieces of several blocks of keys."""
    say("row bits", b)
    q, prefix, cache = make(dev, b, 1, 64, 16, 1, 14000, 40, seed=b)
    n = ints([40] * b, dev)
    want = attention.attention_shared(q, prefix, cache, n)
    for value in (40.0, float("nan")):
        other = q.clone()
        other[0, :, ::3] *= value
        got = attention.attention_shared(other, prefix, cache, n)
        assert torch.equal(got[1:], want[1:]), value
        same = [h for h in range(64) if h % 3]
        assert torch.equal(got[0, :, same], want[0, :, same]), value


@pytest.mark.parametrize("b,s,p", [(130, 1, 40), (12, 24, 12), (60, 1, 3)])
def test_all_requests_on_one_of_many_prefixes(dev, b, s, p):
    """More rows on one prefix than the tiles were chosen for."""
    say("skew", b, s, p)
    q, prefix, cache = make(dev, b, s, 4, 2, p, 150, 30, seed=p)
    share, lengths, plens = [p - 1] * b, [30 - i % 7 for i in range(b)], [150 - i for i in range(p)]
    out = attention.attention_shared(q, prefix, cache, ints(lengths, dev), share=ints(share, dev), prefix_lengths=ints(plens, dev))
    check(out, q, prefix, cache, lengths, share, plens)


def test_what_lies_behind_a_length_is_not_read_into_a_row(dev):
    """NaN in positions past the lengths of prefixes and caches, and in a prefix of other requests."""
    say("nan behind")
    q, prefix, cache = make(dev, 40, 1, 4, 2, 3, 90, 40)
    share, lengths, plens = [i % 2 for i in range(40)], [i for i in range(40)], [50, 33, 90]
    args = dict(share=ints(share, dev), prefix_lengths=ints(plens, dev))
    want = attention.attention_shared(q, prefix, cache, ints(lengths, dev), **args)
    for t, n in zip((prefix, cache), (plens, lengths)):
        for i, size in enumerate(n):
            size = 0 if t is prefix and i == 2 else size
            for codes in (t.k, t.v):
                codes[i, size:].view(torch.uint8).fill_(0x7f)
            for e in (t.k_exponent, t.v_exponent):
                e[i, size:].fill_(255)
    got = attention.attention_shared(q, prefix, cache, ints(lengths, dev), **args)
    assert torch.equal(got, want)


def test_nan_of_one_request_stays_there(dev):
    say("nan request")
    q, prefix, cache = make(dev, 40, 2, 4, 2, 2, 90, 12)
    share = [i % 2 for i in range(40)]
    args = (prefix, cache, ints([12] * 40, dev))
    want = attention.attention_shared(q, *args, share=ints(share, dev))
    q[7, 1, 2] = float("nan")
    cache.v[11].view(torch.uint8)[3].fill_(0x7f)
    prefix.v[1].view(torch.uint8)[80].fill_(0x7f)
    got = attention.attention_shared(q, *args, share=ints(share, dev))
    live = [i for i in range(40) if i % 2 == 0 and i not in (7, 11)]
    assert torch.equal(got[live], want[live]) and got[7, 1, 2].isnan().all() and torch.equal(got[7, 0, 0].isnan(), torch.ones(128, dtype=torch.bool, device=dev))
    assert all(got[i].isnan().all() for i in range(1, 40, 2))


def test_a_prefix_beyond_32_bits(dev):
    """The last prefix starts 4.3 GB into the codes."""
    say("far prefix")
    p, cp, hk = 3, 262144 + 64, 64
    prefix = kv_cache.QuantizedCache(*(torch.zeros(shape, dtype=torch.uint8, device=dev) for shape in
                                       ((p, cp, hk, 128), (p, cp, hk, 4), (p, cp, hk, 128), (p, cp, hk, 4))))
    prefix = kv_cache.QuantizedCache(prefix.k.view(torch.float8_e4m3fn), prefix.k_exponent, prefix.v.view(torch.float8_e4m3fn), prefix.v_exponent)
    g = torch.Generator().manual_seed(1)
    small = filled(dev, g, 1, 100, hk)
    for t, u in zip(prefix, small):
        t[2, :100].view(torch.uint8).copy_(u[0].view(torch.uint8))
        t[2, cp - 100:].view(torch.uint8).copy_(u[0].view(torch.uint8))
    q, cache = bf16_randn(g, (2, 1, hk, 128)).to(dev), filled(dev, g, 2, 4, hk)
    n = ints([4, 2], dev)
    got = attention.attention_shared(q, prefix, cache, n, share=ints([2, 2], dev), prefix_lengths=ints([0, 0, 100], dev))
    check(got, q, small, cache, [4, 2], [0, 0], [100])
    # The zeros in between weigh exp(0): the first and the last keys alone stand out where q is large.
    got = attention.attention_shared(q * 64, prefix, cache, n, share=ints([2, -1], dev), prefix_lengths=ints([0, 0, cp], dev))
    assert got.isfinite().all() and got[0].any()


def test_strides_streams_and_graphs(dev):
    say("graph")
    q, prefix, cache = make(dev, 20, 3, 8, 2, 3, 200, 24)
    fused = torch.zeros(20, 3, 24, 128, dtype=torch.bfloat16, device=dev)
    fused[:, :, 8:16] = q
    share, plens, n = ints([i % 4 - 1 for i in range(20)], dev), ints([200, 11, 77], dev), ints([24 - i for i in range(20)], dev)
    args = dict(share=share, prefix_lengths=plens)
    want = attention.attention_shared(q, prefix, cache, n, **args)
    assert torch.equal(attention.attention_shared(fused[:, :, 8:16], prefix, cache, n, **args), want)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert attention.attention_shared(q, prefix, cache, n, out=out, **args) is out
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)
    graphs, outs = [], []
    for _ in range(2):  # two captured steps whose inputs change between the replays
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(attention.attention_shared(q, prefix, cache, n, **args))
    for i in range(3):
        share.copy_(share.roll(1))
        plens.copy_(plens.roll(1))
        n.copy_(n.roll(3))
        for graph in graphs:
            graph.replay()
        want = attention.attention_shared(q, prefix, cache, n, **args)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want), i


def test_two_graphs_of_one_memory_pool(dev):
    """Captured steps whose workspaces may lie at the same place, replayed in turn with eager calls between."""
    say("two graphs")
    q, prefix, cache = make(dev, 40, 2, 4, 2, 2, 300, 40)
    share, n = ints([i % 3 - 1 for i in range(40)], dev), ints([i for i in range(40)], dev)
    few, one = q[:5].clone(), kv_cache.QuantizedCache(*(t[:1].clone() for t in prefix))
    own, m = kv_cache.QuantizedCache(*(t[:5].clone() for t in cache)), ints([9, 0, 40, 3, 17], dev)
    calls = (lambda: attention.attention_shared(q, prefix, cache, n, share=share), lambda: attention.attention_shared(few, one, own, m))
    for f in calls:
        f()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, f in zip(graphs, calls):
        with torch.cuda.graph(graph, pool=graphs[0].pool() if outs else None):
            outs.append(f())
    for i in range(3):
        q.copy_(torch.randn_like(q.float()).to(torch.bfloat16))
        few.copy_(torch.randn_like(few.float()).to(torch.bfloat16))
        n.add_(1)
        for graph, out, f in zip(graphs, outs, calls):
            graph.replay()
            want = f()
            torch.cuda.synchronize()
            assert torch.equal(out, want), i


def test_agrees_with_attention_over_one_cache(dev):
    """Prefix and own keys in one cache per request, through attention_cached."""
    say("one cache")
    q, prefix, cache = make(dev, 6, 4, 8, 4, 2, 150, 20)
    share = [0, 1, 1, 0, 1, 0]
    plens, n = [150, 99], [20, 4, 11, 9, 20, 5]
    joined = kv_cache.empty_cache(6, 170, 4, 128, dev)
    for i in range(6):
        t = plens[share[i]]
        for dst, a, b in zip(joined, prefix, cache):
            dst[i, :t].view(torch.uint8).copy_(a[share[i], :t].view(torch.uint8))
            dst[i, t:t + n[i]].view(torch.uint8).copy_(b[i, :n[i]].view(torch.uint8))
    tree = random_tree(6, 4, 3).to(dev)
    a = attention.attention_cached(q, joined, ints([plens[share[i]] + n[i] for i in range(6)], dev), tree=tree)
    b = attention.attention_shared(q, prefix, cache, ints(n, dev), share=ints(share, dev), prefix_lengths=ints(plens, dev), tree=tree)
    assert (a.float() - b.float()).abs().max() <= 2.0 ** -8 * a.float().abs().max()   # one rounding each


def test_refusals(dev):
    say("refusals")
    U = _native.Unsupported
    q, prefix, cache = make(dev, 2, 3, 4, 2, 2, 40, 9)
    n, share = ints([9, 9], dev), ints([0, 1], dev)
    sh = attention.attention_shared
    one = kv_cache.QuantizedCache(*(t[:1] for t in prefix))
    for args, kw in (((q, prefix, cache, n), {}), ((q.float(), one, cache, n), {}), ((q[:1], one, cache, n), {}), ((q[..., :64], one, cache, n), {}),
                     ((q, one, cache, n.long()), {}), ((q, one, cache, n[:1]), {}), ((q, one, cache, n.cpu()), {}), ((q, one, cache, [9, 9]), {}),
                     ((q, prefix, cache, n), dict(share=share[:1])), ((q, prefix, cache, n), dict(share=share, prefix_lengths=ints([1], dev))),
                     ((q, one, cache, n), dict(tree=torch.ones(3, 2, dtype=torch.bool, device=dev))),
                     ((q, one, cache, n), dict(tree=torch.ones(3, 3, device=dev))), ((q[:, :, :3], one, cache, n), {}),
                     ((q, filled(dev, torch.Generator(), 1, 4, 4), cache, n), {}),
                     ((torch.zeros(2, 65, 4, 128, dtype=torch.bfloat16, device=dev), one, cache, n), {}),
                     ((q, kv_cache.empty_cache(1, 0, 2, 128, dev), cache, n), {})):
        with pytest.raises(U):
            sh(*args, **kw)
    with pytest.raises(ValueError):
        sh(q, one, cache, n, out=torch.empty_like(q).float())
    with pytest.raises(_native.QimError):
        sh(q, one, cache, n, out=q)
    for scale in (0.0, -1.0, float("nan")):
        with pytest.raises(_native.QimError):
            sh(q, one, cache, n, scale=scale)
    assert sh(q[:, :0], one, cache, n).shape == (2, 0, 4, 128)
