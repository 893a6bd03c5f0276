"""Attention over the MXFP8 cache: how far from float64 it may be -- the output is
rounded to bf16 once, and nothing before it is held in that few bits -- and its masks' bytes."""
import pytest
import torch

from qwen_image_accel.kernels import attention, kv_cache
from tests import requests_ref as R
from tests.helpers import bf16_randn

pytestmark = pytest.mark.gpu


def tight_bound(q, k, v, lengths, tree=None):
    """(o, bound) in float64.  The probability p of a key enters the product with V as two bf16 terms, the second
    the rounding error of the first: HALF^2 of p is left.  A score of D products in fp32 is off by at most D * F32 of
    the sum of their magnitudes (and 2 more roundings), which moves p by that much relative to its size, in
    the numerator and in the sum.  Sums over n keys add at most one F32 of the sum of magnitudes for every key
    (fp32 additions in any order), twice (numerator and sum), exp2 and the join a few more (64).  The
    output is rounded once."""
    want, loose = R.attention(q, k, v, lengths, tree)
    # requests_ref's bound is (HALF + 4 ds + 64 F32) mag + HALF |want|: its magnitudes without p's rounding.
    magnitude, _ = R.attention(q, k, v.abs(), lengths, tree)
    n = lengths.clamp(0, k.shape[1]).double().view(-1, 1, 1, 1)
    inner = loose - R.HALF * want.abs() - R.HALF * magnitude + (R.HALF * R.HALF + 2 * n * R.F32) * magnitude
    return want, (1 + R.HALF) * inner + R.HALF * want.abs()


@pytest.mark.parametrize("b,s,h,hk,c,lengths,drafted", [
    (1, 1, 8, 8, 40, [40], False), (2, 1, 32, 8, 257, [257, 100], False), (2, 24, 4, 4, 500, [500, 47], True),
    (2, 5, 20, 20, 700, [700, 640], False), (1, 40, 8, 4, 300, [300], True)])
def test_only_the_output_is_rounded_to_bf16(dev, b, s, h, hk, c, lengths, drafted):
    print("[case] rounding", b, s, h, hk, c, lengths, drafted, flush=True)
    g = torch.Generator().manual_seed(c)
    q = bf16_randn(g, (b, s, h, 128))
    cache = kv_cache.empty_cache(b, c, hk, 128, dev)
    kv_cache.write_cache(cache, bf16_randn(g, (b, c, hk, 128)).to(dev), bf16_randn(g, (b, c, hk, 128)).to(dev))
    tree = torch.ones(s, s, dtype=torch.bool).tril() if drafted else None
    n = torch.tensor(lengths, dtype=torch.int32)
    out = attention.attention_cached(q.to(dev), cache, n.to(dev), tree=None if tree is None else tree.to(dev))
    want, bound = tight_bound(q, *(t.cpu() for t in kv_cache.read_cache(cache)), n, tree)
    err = (out.double().cpu() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("s", [1, 2, 3, 4, 5, 7, 24, 64])
def test_tree_bytes_other_than_one_are_true(dev, s):
    """A mask of bytes viewed as bool: every byte that is not 0 shows its key, however many tokens there are."""
    print("[case] tree bytes", s, flush=True)
    g = torch.Generator().manual_seed(s)
    q = bf16_randn(g, (2, s, 4, 128)).to(dev)
    cache = kv_cache.empty_cache(2, 90, 2, 128, dev)
    kv_cache.write_cache(cache, bf16_randn(g, (2, 90, 2, 128)).to(dev), bf16_randn(g, (2, 90, 2, 128)).to(dev))
    n = torch.tensor([90, 70], dtype=torch.int32, device=dev)
    values = torch.tensor([0, 0, 0, 1, 2, 64, 128, 254, 255], dtype=torch.uint8)
    tree = values[torch.randint(0, 9, (2, s, s), generator=g)].to(dev)
    want = attention.attention_cached(q, cache, n, tree=tree != 0)
    assert torch.equal(attention.attention_cached(q, cache, n, tree=tree.view(torch.bool)), want)
