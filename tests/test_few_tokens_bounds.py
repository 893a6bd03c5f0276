"""The bounds of the few-token tests notice one lost key, one rounding too many and one wrong code (no GPU: the mistakes are planted in
the oracle)."""
import torch

from tests import few_tokens_bounds as B


def rows(t, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    k, v = ((spread * torch.randn(t, 128, generator=g)).to(torch.bfloat16).double() for _ in range(2))
    return torch.randn(8, 128, generator=g).to(torch.bfloat16).double(), k, v


def outside(got, want, e):
    return bool(((got - want).abs() > B.rounded(want, e)).any())


def test_a_lost_key_is_seen():
    for t in (3, 40, 700, 2000):
        q, k, v = rows(t, t)
        seen = torch.ones(8, t, dtype=torch.bool)
        o, e = B.attention_rows(q, k, v, seen, 128 ** -0.5)
        assert not outside(o.to(torch.bfloat16).double(), o, e)
        for lost in (0, t // 2, t - 1):
            keep = torch.arange(t) != lost
            less, _ = B.attention_rows(q, k[keep], v[keep], seen[:, keep], 128 ** -0.5)
            assert outside(less.to(torch.bfloat16).double(), o, e), (t, lost)


def test_one_rounding_of_p_is_seen():
    """Values that cancel in pairs: p in one bf16 term shows, in two it does not."""
    for t in (2, 6, 60):
        q, k, v = rows(t, t, 0.3)
        v[1::2] = -v[0::2]
        k[1::2] = (k[0::2] + 0.05 * torch.randn(t // 2, 128, generator=torch.Generator().manual_seed(1))).to(torch.bfloat16).double()
        seen = torch.ones(8, t, dtype=torch.bool)
        o, e = B.attention_rows(q, k, v, seen, 128 ** -0.5)
        w = q @ k.T * 128 ** -0.5
        p = torch.exp(w - w.amax(-1, keepdim=True))
        total = p.sum(-1, keepdim=True)
        one = p.to(torch.bfloat16).double()
        two = one + (p - one).to(torch.bfloat16).double()
        assert outside((one @ v / total).to(torch.bfloat16).double(), o, e), t
        assert not outside((two @ v / total).to(torch.bfloat16).double(), o, e), t


def test_a_lost_or_repeated_key_moves_a_count():
    for t in (5, 1000, 12000):
        g = torch.Generator().manual_seed(t)
        v = B.counted(g, (), t).double()
        assert v.sum(0).max() - v.sum(0).min() <= 1 and (v.sum(1) == 1).all()
        want = v.mean(0)
        for other in (torch.cat([v, v[t // 3:t // 3 + 1]]), v[torch.arange(t) != t // 3]):
            got = other.mean(0).to(torch.bfloat16).double()
            assert ((got - want).abs() > B.HALF * want + 8 * B.F32).any(), t


def test_one_wrong_code_is_seen():
    g = torch.Generator().manual_seed(1)
    for k in (128, 4096, 12288):
        codes = torch.randint(0, 256, (16, k // 2), generator=g, dtype=torch.uint8)
        scales, x = torch.rand(16, k // 64, generator=g).to(torch.bfloat16), torch.randn(4, k, generator=g).to(torch.bfloat16)
        y, e = B.four_bit(x, codes, scales, None)
        wrong = codes.clone()
        wrong[:, k // 4] ^= 16
        z, _ = B.four_bit(x, wrong, scales, None)
        assert outside_fp32(z, y, e) and not outside_fp32(y.float().double(), y, e)


def outside_fp32(got, want, e):
    return bool(((got - want).abs() > B.rounded(want, e, torch.float32)).any())
