"""Attention of a few tokens over the MXFP8 cache against float64."""
import pytest
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import attention, kv_cache
from tests import requests_ref as R
from tests.helpers import bf16_randn

pytestmark = pytest.mark.gpu


def say(*a):
    print("[case]", *a, flush=True)


def make(dev, b, s, h, hk, c, seed=0, kscale=1.0):
    g = torch.Generator().manual_seed(seed)
    q = bf16_randn(g, (b, s, h, 128)).to(dev)
    cache = kv_cache.empty_cache(b, c, hk, 128, dev)
    kv_cache.write_cache(cache, bf16_randn(g, (b, c, hk, 128), kscale).to(dev), bf16_randn(g, (b, c, hk, 128)).to(dev))
    return q, cache


def lens(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def check(out, q, cache, lengths, tree=None, scale=None):
    k, v = kv_cache.read_cache(cache)
    want, bound = R.attention(q, k, v, lengths.cpu(), tree, scale)
    err = (out.double().cpu() - want).abs()
    worst = float((err / bound.clamp(min=1e-30)).max())
    assert out.isfinite().all() and (err <= bound).all(), worst


def random_tree(b, s, seed):
    g = torch.Generator().manual_seed(seed)
    m = torch.zeros(b, s, s, dtype=torch.bool)
    for i in range(b):
        for j in range(s):
            if j:
                m[i, j] = m[i, int(torch.randint(0, j, (1,), generator=g))]
            m[i, j, j] = True
    return m


@pytest.mark.parametrize("b,s,h,hk,c,lengths", [
    (1, 1, 1, 1, 1, [1]), (1, 1, 2, 2, 33, [33]), (4, 1, 2, 2, 70, [0, 1, 31, 32]), (4, 1, 4, 1, 70, [63, 64, 65, 70]),
    (2, 1, 32, 8, 257, [257, 100]), (1, 3, 6, 2, 129, [128]), (2, 16, 4, 2, 300, [300, 17]), (1, 33, 2, 2, 200, [199]),
    (1, 64, 2, 1, 190, [190]), (2, 64, 8, 2, 100, [64, 100]), (3, 2, 40, 1, 96, [96, 5, 2]), (1, 1, 3, 3, 5000, [4999]),
    (2, 5, 20, 20, 1111, [1111, 640]), (1, 1, 8, 8, 20000, [20000])])
def test_against_float64(dev, b, s, h, hk, c, lengths):
    say("attention", b, s, h, hk, c, lengths)
    q, cache = make(dev, b, s, h, hk, c, seed=s + c)
    n = lens(lengths, dev)
    check(attention.attention_cached(q, cache, n), q, cache, n)


@pytest.mark.parametrize("b,s,h,hk,c,lengths,shared", [
    (1, 2, 1, 1, 2, [2], False), (3, 5, 2, 2, 60, [5, 33, 60], False), (2, 24, 4, 4, 500, [500, 47], False),
    (2, 64, 2, 1, 150, [64, 150], False), (1, 33, 8, 2, 97, [97], True), (2, 7, 4, 2, 40, [3, 0], False),
    (2, 63, 1, 1, 700, [700, 320], True)])
def test_tree(dev, b, s, h, hk, c, lengths, shared):
    """Tree masks of one per sequence and shared, the tree inside one block, over several, and longer than
    the sequence (keys before position 0 do not exist)."""
    say("tree", b, s, h, hk, c, lengths, shared)
    q, cache = make(dev, b, s, h, hk, c, seed=s + c)
    tree = random_tree(b, s, s)
    tree = tree[0].contiguous() if shared else tree
    n = lens(lengths, dev)
    check(attention.attention_cached(q, cache, n, tree=tree.to(dev)), q, cache, n, tree)


@pytest.mark.parametrize("b,c", [(70, 600), (130, 1000), (300, 90)])
def test_batches_of_many_unequal_sequences(dev, b, c):
    """More sequences than a wave has lanes, of lengths from 0 to all, in chunks or one each."""
    say("many sequences", b, c)
    q, cache = make(dev, b, 1, 2, 2, c, seed=b)
    n = torch.randint(0, c + 1, (b,), generator=torch.Generator().manual_seed(c), dtype=torch.int32)
    n[::9], n[1], n[-1] = 0, c, c - 31
    n = n.to(dev)
    check(attention.attention_cached(q, cache, n), q, cache, n)


def test_long_cache_with_more_rows_than_a_tile(dev):
    say("tiles of 32 rows, chunks")
    b, s, c = 5, 40, 8000
    q, cache = make(dev, b, s, 8, 8, c)
    tree, n = random_tree(b, s, 3), lens([3001, 100, 33, 40, 0], dev)
    check(attention.attention_cached(q, cache, n, tree=tree.to(dev)), q, cache, n, tree)


def test_out_over_q_is_refused(dev):
    say("out over q")
    q, cache = make(dev, 2, 3, 2, 2, 64)
    with pytest.raises(_native.QimError, match="overlaps"):
        attention.attention_cached(q, cache, lens([64, 5], dev), out=q)


def test_causal_equals_one_token_at_a_time(dev):
    """A causal tree over the last S tokens gives what S single-token calls of growing length give."""
    say("causal vs single tokens")
    b, s, h, hk, c = 2, 12, 8, 4, 300
    q, cache = make(dev, b, s, h, hk, c)
    n = lens([300, 177], dev)
    causal = torch.ones(s, s, dtype=torch.bool, device=dev).tril()
    got = attention.attention_cached(q, cache, n, tree=causal)
    check(got, q, cache, n, causal)
    for i in range(s):
        m = n - (s - 1 - i)
        check(attention.attention_cached(q[:, i:i + 1], cache, m), q[:, i:i + 1], cache, m)


def test_rows_that_see_nothing_are_zeros(dev):
    say("empty rows")
    q, cache = make(dev, 3, 4, 2, 2, 64)
    tree = torch.ones(3, 4, 4, dtype=torch.bool, device=dev)
    tree[0, 2] = False                         # of a sequence whose keys are all drafted
    n = lens([4, 0, -7], dev)
    out = attention.attention_cached(q, cache, n, tree=tree)
    assert not out[0, 2].any() and not out[1].any() and not out[2].any()
    assert out[0, 0].any()
    check(out, q, cache, n, tree)


def test_lengths_outside_the_cache_count_as_its_ends(dev):
    say("lengths clamp")
    q, cache = make(dev, 2, 1, 2, 2, 50)
    assert torch.equal(attention.attention_cached(q, cache, lens([2 ** 31 - 1, 51], dev)),
                       attention.attention_cached(q, cache, lens([50, 50], dev)))


@pytest.mark.parametrize("length", [0, 5, 32, 37, 64])
def test_what_lies_behind_the_length_is_not_read_into_the_result(dev, length):
    say("garbage behind", length)
    q, cache = make(dev, 1, 2, 4, 2, 96)
    n = lens([length], dev)
    want = attention.attention_cached(q, cache, n)
    for byte in (0x7f, 0xff, 0x7e):            # NaN codes, the largest code
        for t in (cache.k, cache.v):
            t.view(torch.uint8)[:, length:] = byte
        for t in (cache.k_exponent, cache.v_exponent):
            t[:, length:] = 254
        assert torch.equal(attention.attention_cached(q, cache, n), want)


@pytest.mark.parametrize("g", [1, 4])
def test_not_finite_values_stay_with_the_rows_that_see_them(dev, g):
    """NaN in K or V of one drafted branch: the rows of the other branch do not change."""
    say("NaN in a branch", g)
    b, s, hk, c = 1, 40, 2, 90
    q, cache = make(dev, b, s, hk * g, hk, c)
    tree = torch.zeros(s, s, dtype=torch.bool)
    for i in range(s):                         # two chains: even and odd tokens
        tree[i, i % 2:i + 1:2] = True
    tree, n = tree.to(dev), lens([80], dev)
    want = attention.attention_cached(q, cache, n, tree=tree)
    for t in (cache.v, cache.k):
        keep = t.clone()
        t.view(torch.uint8)[0, 80 - s + 7, 1, 3] = 0x7f      # drafted token 7, the odd chain
        out = attention.attention_cached(q, cache, n, tree=tree)
        even, odd = torch.arange(0, s, 2, device=dev), torch.arange(7, s, 2, device=dev)
        assert torch.equal(out[:, even], want[:, even])
        assert torch.equal(out[:, 1:7:2], want[:, 1:7:2])
        assert torch.equal(out[:, :, :g], want[:, :, :g])    # the other K/V head
        bad = torch.isnan(out[0, odd, g:])
        assert bad[..., 3].all() if t is cache.v else bad.all()
        if t is cache.v:
            other = [d for d in range(128) if d != 3]
            assert torch.equal(out[0, odd][:, g:, other], want[0, odd][:, g:, other])
        t.copy_(keep)


def test_nan_in_a_query_stays_in_its_row(dev):
    say("NaN in q")
    q, cache = make(dev, 2, 3, 4, 2, 70)
    n = lens([70, 31], dev)
    want = attention.attention_cached(q, cache, n)
    q[1, 1, 2, 5] = float("nan")
    out = attention.attention_cached(q, cache, n)
    assert torch.isnan(out[1, 1, 2]).all()
    out[1, 1, 2] = want[1, 1, 2]
    assert torch.equal(out, want)


def test_large_scores_and_late_maximum(dev):
    """Scores of several hundred, the largest key last: the running maximum moves far."""
    say("large scores")
    q, cache = make(dev, 1, 4, 4, 4, 400, kscale=8.0)
    k, v = kv_cache.read_cache(cache)
    k[:, 399] = q[:, 0] * 4
    kv_cache.write_cache(cache, k, v)
    n = lens([400], dev)
    check(attention.attention_cached(q * 4, cache, n), q * 4, cache, n)
    check(attention.attention_cached(q, cache, n, scale=1.5), q, cache, n, scale=1.5)


def test_strided_queries_and_out(dev):
    say("strided q")
    q, cache = make(dev, 3, 5, 4, 2, 64)
    n = lens([64, 9, 33], dev)
    want = attention.attention_cached(q, cache, n)
    wide = torch.empty(3, 7, 3, 4, 128, dtype=torch.bfloat16, device=dev)
    wide[:, 1:6, 2] = q
    out = torch.full_like(q, 7.0)
    assert attention.attention_cached(wide[:, 1:6, 2], cache, n, out=out) is out
    assert torch.equal(out, want)
    assert attention.attention_cached(q[:, :0], cache, n).shape == (3, 0, 4, 128)


def test_repeats_are_identical(dev):
    say("repeat")
    q, cache = make(dev, 2, 2, 8, 8, 3000)
    n = lens([3000, 1234], dev)
    first = attention.attention_cached(q, cache, n)
    for _ in range(3):
        assert torch.equal(attention.attention_cached(q, cache, n), first)


def test_offsets_past_32_bits(dev):
    """More than 2^32 code bytes per tensor: keys of zeros, and the last three positions that decide the
    result."""
    h, d = 4, 128
    c = (1 << 32) // (h * d) + 700
    say("cache attention > 4 GiB", c)
    g = torch.Generator().manual_seed(1)
    cache = kv_cache.empty_cache(1, c, h, d, dev)
    for t in cache:
        t.view(torch.uint8).zero_()
    q = bf16_randn(g, (1, 1, h, d), 4.0).to(dev)
    k, v = (q * 8).expand(1, 3, h, d).contiguous(), bf16_randn(g, (1, 3, h, d)).to(dev)
    kv_cache.write_cache(cache, k, v, start=c - 3)
    out = attention.attention_cached(q, cache, lens([c], dev))
    # p of a zero key is exp(-|q|^2 * 8 / sqrt(128)), |q|^2 about 2000: nothing beside 8 million keys
    small = kv_cache.empty_cache(1, 3, h, d, dev)
    kv_cache.write_cache(small, k, v)
    check(out, q, small, lens([3], dev))
