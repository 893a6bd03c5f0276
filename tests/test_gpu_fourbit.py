"""Products of few rows with 4-bit weights against float64."""
import pytest
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import fourbit
from tests import few_tokens_ref as R
from tests.helpers import bf16_randn

pytestmark = pytest.mark.gpu

KINDS = [("int4", 32, True), ("int4", 64, True), ("int4", 128, True), ("int4", 32, False), ("int4", 128, False), ("mxfp4", 32, False)]


def say(*a):
    print("[case]", *a, flush=True)


def random_weight(dev, n, k, kind, group, zeros, seed=0):
    """Any codes, scales of several octaves, any zero points: not only what a quantizer makes."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    if kind == "mxfp4":
        scales = torch.randint(112, 122, (n, k // 32), generator=g, dtype=torch.uint8)
    else:
        scales = (torch.rand(n, k // group, generator=g) * 0.02 - 0.001).to(torch.bfloat16)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    return tuple(None if t is None else t.to(dev) for t in (codes, scales, z))


def pack(raw):
    return fourbit.pack_weight(raw[0], raw[1], zeros=raw[2])


def check(got, want, error):
    bound = R.rounded(want, error, got.dtype)
    err = (got.reshape(want.shape).double().cpu() - want).abs()
    assert got.isfinite().all() and (err <= bound).all(), float((err / bound).max())


SIZES = [(1, 1, 128), (1, 16, 256), (2, 17, 384), (5, 100, 1024), (16, 48, 4096), (17, 33, 640), (31, 250, 512), (33, 64, 2176),
         (64, 512, 1024), (65, 30, 256), (100, 130, 1536), (257, 96, 512), (3, 4096, 4096), (1, 1001, 12288)]


@pytest.mark.parametrize("kind,group,zeros", KINDS)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(dev, m, n, k, kind, group, zeros):
    say("four bits", m, n, k, kind, group, zeros)
    raw = random_weight(dev, n, k, kind, group, zeros, seed=m + n)
    x = bf16_randn(torch.Generator().manual_seed(k), (m, k)).to(dev)
    y, e = R.four_bit(x, *raw)
    check(fourbit.matmul(x, pack(raw)), y, e)
    check(fourbit.matmul(x, pack(raw), dtype=torch.float32), y, e)


@pytest.mark.parametrize("kind,group,k", [("int4", 32, 32), ("int4", 32, 96), ("int4", 32, 160), ("int4", 64, 64), ("int4", 64, 192),
                                          ("int4", 64, 1088), ("mxfp4", 32, 32), ("mxfp4", 32, 992)])
@pytest.mark.parametrize("m", [1, 20, 90])
def test_a_width_that_ends_inside_a_step(dev, m, kind, group, k):
    say("short steps", m, kind, group, k)
    raw = random_weight(dev, 40, k, kind, group, kind == "int4", seed=k)
    wide = torch.full((m, k + 64), float("nan"), dtype=torch.bfloat16, device=dev)   # what lies behind a row is not read
    x = wide[:, :k]
    x.copy_(bf16_randn(torch.Generator().manual_seed(k), (m, k)))
    y, e = R.four_bit(x, *raw)
    check(fourbit.matmul(x, pack(raw)), y, e)


@pytest.mark.parametrize("kind,group,zeros", KINDS)
@pytest.mark.parametrize("m,n,k", [(1, 16, 128), (4, 75, 640), (16, 256, 4096), (24, 130, 1024), (40, 64, 512), (130, 96, 768)])
def test_swiglu(dev, m, n, k, kind, group, zeros):
    say("swiglu", m, n, k, kind, group, zeros)
    a, b = (random_weight(dev, n, k, kind, group, zeros, seed=s) for s in (1, 2))
    x = bf16_randn(torch.Generator().manual_seed(k), (m, k), 0.3).to(dev)
    y, e = R.swiglu(R.four_bit(x, *a), R.four_bit(x, *b))
    check(fourbit.swiglu(x, pack(a), pack(b)), y, e)


# Rows and columns of a plain product (of a SwiGLU: half the columns) for each height of the shared tiles (16, 32, 64, 80 and
# 128 rows) and, for int4, each of their widths.
TILES = [(15, 65530), (30, 24600), (30, 14210), (48, 12200), (40, 24610), (100, 8100), (150, 8100), (70, 20000), (200, 8390), (1020, 4090)]


@pytest.mark.parametrize("kind,group,k", [("int4", 32, 160), ("int4", 64, 192), ("int4", 128, 384), ("mxfp4", 32, 224)])
@pytest.mark.parametrize("m,n", TILES)
def test_many_columns(dev, m, n, kind, group, k):
    say("many columns", m, n, k, kind, group)
    raw = random_weight(dev, n, k, kind, group, kind == "int4", seed=m)
    x = bf16_randn(torch.Generator().manual_seed(k), (m, k)).to(dev)
    bias = bf16_randn(torch.Generator().manual_seed(1), (n,)).to(dev)
    w = pack(raw)
    check(fourbit.matmul(x, w, bias=bias), *R.four_bit(x, *raw, bias=bias))
    a, b = (tuple(None if t is None else t[h::2].contiguous() for t in raw) for h in (0, 1))
    x = 0.3 * x
    check(fourbit.swiglu(x, pack(a), pack(b)), *R.swiglu(R.four_bit(x, *a), R.four_bit(x, *b)))


def test_every_code(dev):
    """A weight of each code alone, times powers of two: exact."""
    say("every code")
    for kind in ("int4", "mxfp4"):
        for code in range(16):
            codes = torch.full((16, 64), code * 17, dtype=torch.uint8, device=dev)
            if kind == "int4":
                scales, z = torch.full((16, 1), 0.5, dtype=torch.bfloat16, device=dev), torch.arange(16, dtype=torch.uint8, device=dev)[:, None]
                want = (code - torch.arange(16.0)) * 0.5
            else:
                exponents = torch.arange(16, device=dev)[:, None].expand(16, 4) + 119
                scales, z = exponents.to(torch.uint8).contiguous(), None
                want = (fourbit.E2M1[code & 7] * (-1 if code > 7 else 1)) * torch.exp2(torch.arange(16.0) - 8)
            x = torch.zeros(128, 128, dtype=torch.bfloat16, device=dev).fill_diagonal_(4.0)
            got = fourbit.matmul(x, fourbit.pack_weight(codes, scales, zeros=z), dtype=torch.float32)
            assert torch.equal(got.cpu(), (4 * want).expand(128, 16)), (kind, code)


@pytest.mark.parametrize("kind,group,zeros", [("int4", 64, True), ("int4", 128, False), ("mxfp4", 32, False)])
def test_infinities_and_nan_stay_in_their_rows(dev, kind, group, zeros):
    """Rows of one tile: one holds infinities, one NaN, one values whose sums with the codes alone leave fp32."""
    say("not finite", kind)
    n, k = 50, 512
    raw = random_weight(dev, n, k, kind, group, zeros, seed=3)
    w = fourbit.dequantize_weight(pack(raw)).double().cpu()
    for m in (7, 40, 90):
        x = bf16_randn(torch.Generator().manual_seed(m), (m, k)).to(dev)
        want = fourbit.matmul(x, pack(raw))
        x[1, 100] = float("inf")
        x[2, 7], x[2, 300] = float("-inf"), float("nan")
        x[3] = 0
        x[3, :group:2] = 1.5 * 2.0 ** 120 if group == 64 else 2.0 ** 120
        got = fourbit.matmul(x, pack(raw))
        live = torch.tensor([i not in (1, 2, 3) for i in range(m)], device=dev)
        check(got[live], *R.four_bit(x[live], *raw))
        assert torch.equal(got[live], want[live])
        exact = x.double().cpu() @ w.T
        assert got[2].isnan().all()
        hot = w[:, 100]
        assert torch.equal(got[1].cpu().double()[hot > 0], exact[1][hot > 0]) and torch.equal(got[1].cpu().double()[hot < 0], exact[1][hot < 0])
        assert got[1].cpu()[hot == 0].isnan().all()
        per = (w / fourbit.unpack_weight(pack(raw))[1].double().cpu().repeat_interleave(group, 1) if kind == "int4" else w) * x[3].double().cpu()
        fits = (per.unflatten(1, (-1, group)).sum(-1).abs() < 2.0 ** 127).all(1)   # every group's own sum is in fp32
        err = (got[3].cpu().double() - exact[3]).abs()[fits]
        assert fits.any() and (err <= R.rounded(*R.four_bit(x[3:4], *raw))[0][fits]).all()


def test_rows_layouts_and_out(dev):
    say("layouts")
    raw = random_weight(dev, 75, 256, "int4", 64, True)
    w, bias = pack(raw), bf16_randn(torch.Generator().manual_seed(1), (75,)).to(dev)
    wide = torch.randn(3, 5, 2 * 256 + 8, device=dev).to(torch.bfloat16)
    x = wide[..., 256:512]
    y, e = R.four_bit(x.reshape(15, 256), *raw, bias=bias)
    got = fourbit.matmul(x, w, bias=bias)
    assert got.shape == (3, 5, 75)
    check(got, y, e)
    for dtype in (torch.bfloat16, torch.float32):
        for pad, first in ((5, 1), (5, 0), (9, 4)):
            big = torch.full((3, 5, 75 + pad), 3.0, dtype=dtype, device=dev)
            out = big[..., first:first + 75]
            assert fourbit.matmul(x, w, bias=bias, out=out, dtype=dtype) is out
            check(out, y, e)
            assert (big[..., :first] == 3).all() and (big[..., first + 75:] == 3).all()
    assert fourbit.matmul(x[:0], w).shape == (0, 5, 75)
    one = fourbit.matmul(x[1, 2:3], w, bias=bias)
    check(one, y[7:8], e[7:8])


def test_same_bits_every_time_and_beside_other_rows(dev):
    """No atomics: the same call gives the same bits; a row's bits do not depend on the other rows' values."""
    say("repeat")
    raw = random_weight(dev, 200, 1024, "int4", 64, True)
    x = bf16_randn(torch.Generator().manual_seed(1), (24, 1024)).to(dev)
    w = pack(raw)
    first = fourbit.matmul(x, w)
    other = x.clone()
    other[5:] = 100 * other[5:].flip(0)
    assert torch.equal(fourbit.matmul(x, w), first) and torch.equal(fourbit.matmul(other, w)[:5], first[:5])


def test_streams_and_graphs(dev):
    say("graph")
    raw = random_weight(dev, 512, 1024, "int4", 128, False)
    w, x = pack(raw), bf16_randn(torch.Generator().manual_seed(1), (4, 1024)).to(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = fourbit.swiglu(x, w, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, fourbit.swiglu(x, w, w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fourbit.matmul(x, w)
    for i in range(3):
        x.copy_(torch.randn_like(x.float()).to(torch.bfloat16))
        graph.replay()
        want = fourbit.matmul(x, w)
        torch.cuda.synchronize()
        assert torch.equal(got, want), i


def test_refusals(dev):
    say("refusals")
    U = _native.Unsupported
    raw = random_weight(dev, 32, 256, "int4", 64, True)
    w, x = pack(raw), torch.zeros(4, 256, dtype=torch.bfloat16, device=dev)
    bf = dict(dtype=torch.bfloat16, device=dev)
    for args, kw in (((x.float(), w), {}), ((x[:, :128], w), {}), ((x.cpu(), w), {}), ((torch.zeros(4, 260, **bf)[:, :256], w), {}),
                     ((torch.zeros(4 * 256 + 1, **bf)[1:].view(4, 256), w), {}), ((x, w), dict(bias=torch.zeros(31, **bf))),
                     ((x, w), dict(bias=torch.zeros(32, device=dev))), ((x, w), dict(out=torch.zeros(4, 31, **bf))),
                     ((x, w), dict(dtype=torch.float16)), ((x, w), dict(out=torch.zeros(4, 32, device=dev))),
                     ((x, w._replace(codes=w.codes.cpu())), {}), ((x, w._replace(zeros=w.zeros[:1])), {}),
                     ((x, w._replace(rows=33)), {}), ((x, w._replace(group=32)), {}), ((x, w._replace(scales=w.scales.float())), {})):
        with pytest.raises(U):
            fourbit.matmul(*args, **kw)
    other = pack(random_weight(dev, 32, 256, "int4", 64, False))
    with pytest.raises(U):
        fourbit.swiglu(x, w, other)
    with pytest.raises(U):
        fourbit.swiglu(x, w, pack(random_weight(dev, 16, 256, "int4", 64, True)))
    wide = torch.zeros(4, 512, **bf)
    with pytest.raises(_native.QimError):
        fourbit.matmul(wide[:, :256], w, out=wide[:, 240:272])
