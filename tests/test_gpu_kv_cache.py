"""The MXFP8 K/V cache: what is written and read back, bit for bit; where it is
written; and the fused pack in front of a step's keys."""
import types

import pytest
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import attention, kv_cache, mxfp8
from tests import requests_ref as R
from tests.helpers import bf16_randn

pytestmark = pytest.mark.gpu


def say(*a):
    print("[case]", *a, flush=True)


def filled(b, c, h, d, dev, byte=0x38):
    cache = kv_cache.empty_cache(b, c, h, d, dev)
    for t in cache:
        t.view(torch.uint8).fill_(byte)
    return cache


@pytest.mark.parametrize("b,s,h,d", [(1, 1, 1, 32), (2, 5, 3, 64), (1, 300, 4, 128), (3, 17, 20, 128), (2, 9, 1, 256),
                                     (1, 2, 5, 96), (1, 1025, 32, 128)])
def test_written_values_read_back(dev, b, s, h, d):
    say("cache values", b, s, h, d)
    g = torch.Generator().manual_seed(b * 1000 + s)
    k = bf16_randn(g, (b, s, h, d), 3.0)
    v = bf16_randn(g, (b, s, h, d)) * (2.0 ** torch.randint(-20, 20, (b, s, h, 1), generator=g)).bfloat16()
    k.view(-1)[:32] = 0                       # a block of zeros
    cache = kv_cache.empty_cache(b, s, h, d, dev)
    kv_cache.write_cache(cache, k.to(dev), v.to(dev))
    for got, x in zip(kv_cache.read_cache(cache), (k, v)):
        assert torch.equal(got.double().cpu(), R.block_values(x))


def test_codes_are_those_of_quantize(dev):
    """Infinities, NaN, the largest and smallest magnitudes among them."""
    say("cache codes vs quantize")
    g = torch.Generator().manual_seed(3)
    x = bf16_randn(g, (1, 64, 4, 128))
    f = x.view(-1)
    big, tiny = torch.finfo(torch.bfloat16).max, 2.0 ** -133
    for i, val in enumerate((big, -big, float("inf"), float("nan"), tiny, -3 * tiny, 448.0, 464.0, 449.0, 2.0 ** -126)):
        f[64 * i:64 * i + 32] *= 0 if abs(val) < 1 else 1
        f[64 * i + i] = val
    cache = kv_cache.empty_cache(1, 64, 4, 128, dev)
    kv_cache.write_cache(cache, x.to(dev), x.to(dev))
    q = mxfp8.quantize(x.view(64, 512).to(dev))
    from tests.helpers import unswizzle_scales
    want = q.values[:64].view(torch.uint8).cpu()
    exps = unswizzle_scales(q.scales.view(torch.uint8).cpu().numpy(), 128, 512)[:64]
    for codes, e in ((cache.k, cache.k_exponent), (cache.v, cache.v_exponent)):
        assert torch.equal(codes.view(torch.uint8).cpu().view(64, 512), want)
        assert (e.cpu().view(64, 16).numpy() == exps).all()


@pytest.mark.parametrize("e", [0, 1, 2, 127, 246, 247, 254])
def test_every_code_reads_back_exactly(dev, e):
    """All 256 codes at the ends of the exponents' range: what bf16 cannot hold (below half its smallest step, or
    above its largest value) rounds as a conversion does; everything a bf16 input can have given is exact."""
    say("read codes, exponent", e)
    cache = filled(1, 8, 1, 32, dev, 0)
    codes = torch.arange(256, dtype=torch.uint8).view(1, 8, 1, 32)
    cache.k.view(torch.uint8).copy_(codes)
    cache.k_exponent.fill_(e)
    got = kv_cache.read_cache(cache)[0].double().cpu().view(-1)
    value = codes.view(torch.float8_e4m3fn).double().view(-1) * 2.0 ** (e - 127)
    exact = value.to(torch.bfloat16).double() == value
    # At e = 254 the unit is 2^127 and bf16 ends below 2^128: the codes below 2.0, 64 of each sign.
    assert exact.sum() >= 128
    assert torch.equal(got[exact], value[exact])
    assert torch.isnan(got[[127, 255]]).all()


@pytest.mark.parametrize("form", ["int", "tensor", "count"])
def test_places(dev, form):
    """Rows go where they are told to; everything else keeps its bytes, rows outside the cache too."""
    say("cache places", form)
    b, s, c, h, d = 4, 6, 16, 3, 64
    g = torch.Generator().manual_seed(11)
    k, v = bf16_randn(g, (b, s, h, d)).to(dev), bf16_randn(g, (b, s, h, d)).to(dev)
    full = kv_cache.empty_cache(b, s, h, d, dev)
    kv_cache.write_cache(full, k, v)
    cache = filled(b, c, h, d, dev)
    want = [t.view(torch.uint8).clone() for t in cache]
    starts, counts = [10] * b, [s] * b
    kw = {"start": 10}
    if form != "int":
        starts = [0, 13, -3, 2 ** 31 - 4]    # whole, past the end, before the start, far outside
        kw["start"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    if form == "count":
        counts = [0, 2, 100, -1]
        kw["count"] = torch.tensor(counts, dtype=torch.int32, device=dev)
    kv_cache.write_cache(cache, k, v, **kw)
    for i in range(b):
        for row in range(min(s, max(0, counts[i]))):
            if 0 <= starts[i] + row < c:
                for w, f in zip(want, full):
                    w[i, starts[i] + row] = f.view(torch.uint8)[i, row]
    for w, t in zip(want, cache):
        assert torch.equal(w, t.view(torch.uint8))


def test_strided_rows_and_batches(dev):
    say("cache strides")
    g = torch.Generator().manual_seed(5)
    b, s, h, d = 3, 7, 2, 64
    fused = bf16_randn(g, (b, s + 2, 3, h, d)).to(dev)
    k, v = fused[:, 1:s + 1, 1], fused[:, 2:, 2]
    cache, plain = kv_cache.empty_cache(b, s, h, d, dev), kv_cache.empty_cache(b, s, h, d, dev)
    kv_cache.write_cache(cache, k, v)
    kv_cache.write_cache(plain, k.contiguous(), v.contiguous())
    for x, y in zip(cache, plain):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    one = k[:1].expand(b, s, h, d)            # one prompt for several sequences
    kv_cache.write_cache(cache, one, v)
    kv_cache.write_cache(plain, one.contiguous(), v.contiguous())
    for x, y in zip(cache, plain):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_read_part_and_nothing(dev):
    say("cache read part")
    g = torch.Generator().manual_seed(6)
    k, v = bf16_randn(g, (2, 9, 3, 128)).to(dev), bf16_randn(g, (2, 9, 3, 128)).to(dev)
    cache = kv_cache.empty_cache(2, 9, 3, 128, dev)
    kv_cache.write_cache(cache, k, v)
    whole = kv_cache.read_cache(cache)
    for rows in (0, 1, 4, 9):
        for part, w in zip(kv_cache.read_cache(cache, rows), whole):
            assert part.shape == (2, rows, 3, 128) and torch.equal(part, w[:, :rows])
    kv_cache.write_cache(cache, k[:, :0], v[:, :0])
    for w, t in zip(whole, kv_cache.read_cache(cache)):
        assert torch.equal(w, t)


def test_offsets_past_32_bits(dev):
    """A cache of more than 2^32 code bytes per tensor: its last positions."""
    h, d = 8, 128
    c = (1 << 32) // (h * d) + 1000
    say("cache > 4 GiB", c)
    g = torch.Generator().manual_seed(7)
    k, v = bf16_randn(g, (1, 3, h, d)).to(dev), bf16_randn(g, (1, 3, h, d)).to(dev)
    cache = filled(1, c, h, d, dev, 0)
    kv_cache.write_cache(cache, k, v, start=torch.tensor([c - 3], dtype=torch.int32, device=dev))
    for got, x in zip(kv_cache.read_cache(cache), (k, v)):
        assert torch.equal(got[:, c - 3:].double().cpu(), R.block_values(x.cpu()))
        assert not got[0, (c - 2000):c - 3].any()


@pytest.mark.parametrize("b,s,p,h,d,view", [(1, 5, 1, 2, 64, False), (2, 33, 7, 3, 128, True), (1, 64, 200, 20, 128, True),
                                            (2, 17, 40, 5, 256, False), (1, 300, 77, 32, 128, True)])
def test_pack(dev, b, s, p, h, d, view):
    """The prefix and v are copied exactly; q and k against float64, rounded once.

    The bound: the mean of squares and its root in fp32 (a few roundings), two products, and per rotated value two
    products and a sum: 16 fp32 roundings of |x cos| + |x' sin| in all, then half a bf16 step."""
    say("pack", b, s, p, h, d, view)
    g = torch.Generator().manual_seed(s)
    qkv = bf16_randn(g, (b, s, 3, h, d)).to(dev)
    q, k, v = qkv.unbind(2) if view else (qkv[:, :, i].contiguous() for i in range(3))
    norms = [types.SimpleNamespace(weight=bf16_randn(g, (d,)).to(dev), eps=1e-6, bias=None) for _ in range(2)]
    freqs = torch.polar(torch.ones(s, d // 2), torch.randn(s, d // 2, generator=g)).to(dev)
    cache = filled(b, p + 3, h, d, dev)
    kv_cache.write_cache(cache, bf16_randn(g, (b, p, h, d)).to(dev), bf16_randn(g, (b, p, h, d)).to(dev))
    before = _native.calls.get("qim_qk_norm_rope_pack_cached", 0)
    oq, ok, ov = attention.prepare_attention_inputs_quantized(q, k, v, *norms, freqs, cache, prefix=p)
    assert _native.calls["qim_qk_norm_rope_pack_cached"] == before + 1
    ck, cv = kv_cache.read_cache(cache, p)
    assert torch.equal(ok[:, :p], ck) and torch.equal(ov, torch.cat([cv, v], 1))
    for got, x, norm in ((oq, q, norms[0]), (ok[:, p:], k, norms[1])):
        x = x.double()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + norm.eps) * norm.weight.double()
        z = torch.complex(x[..., 0::2], x[..., 1::2])
        f = freqs.to(torch.complex128)[None, :, None]
        want = torch.view_as_real(z * f).flatten(-2)
        mag = torch.stack([z.real.abs() * f.real.abs() + z.imag.abs() * f.imag.abs(),
                           z.real.abs() * f.imag.abs() + z.imag.abs() * f.real.abs()], -1).flatten(-2)
        assert ((got.double() - want).abs() <= R.HALF * want.abs() + (1 + R.HALF) * 16 * R.F32 * mag).all()


def test_pack_without_a_prefix(dev):
    """No positions of a cache, or a cache of none: the step's own rows, the same values."""
    say("pack, no prefix")
    g = torch.Generator().manual_seed(3)
    q, k, v = (bf16_randn(g, (2, 9, 3, 128)).to(dev) for _ in range(3))
    norms = [types.SimpleNamespace(weight=bf16_randn(g, (128,)).to(dev), eps=1e-6, bias=None) for _ in range(2)]
    freqs = torch.polar(torch.ones(9, 64), torch.randn(9, 64, generator=g)).to(dev)
    some = attention.prepare_attention_inputs_quantized(q, k, v, *norms, freqs, filled(2, 4, 3, 128, dev), prefix=0)
    none = attention.prepare_attention_inputs_quantized(q, k, v, *norms, freqs, kv_cache.empty_cache(2, 0, 3, 128, dev))
    whole = attention.prepare_attention_inputs_quantized(q, k, v, *norms, freqs, filled(2, 4, 3, 128, dev))
    for a, b, c, skip in zip(some, none, whole, (0, 4, 4)):
        assert torch.equal(a, b) and torch.equal(a, c[:, skip:])
    assert torch.equal(some[2], v)
