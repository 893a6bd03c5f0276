"""Low-rank adapters of several requests against float64."""
import pytest
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import adapters
from tests import requests_ref as R
from tests.helpers import bf16_randn

pytestmark = pytest.mark.gpu


def say(*a):
    print("[case]", *a, flush=True)


def make(dev, m, k, n, r, a, parts=1, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (bf16_randn(g, (m, k)).to(dev), bf16_randn(g, (a, parts * r, k), k ** -0.5).to(dev),
            bf16_randn(g, (a, n, r), r ** -0.5).to(dev), (torch.rand(a, generator=g) + 0.5).to(dev),
            bf16_randn(g, (m, n)).to(dev), torch.randint(-1, a, (m,), generator=g, dtype=torch.int32).to(dev))


def check(out, *args, **kw):
    want, bound = R.low_rank(*args, **kw)
    err = (out.double().reshape(want.shape) - want).abs()
    assert out.isfinite().all() and (err <= bound).all(), float((err / bound.clamp(min=1e-30)).max())


@pytest.mark.parametrize("m,k,n,r,a,parts", [
    (1, 8, 8, 8, 1, 1), (1, 4096, 4096, 16, 3, 1), (16, 256, 512, 16, 16, 1), (17, 264, 40, 8, 5, 1), (33, 1000, 96, 24, 2, 3),
    (5, 128, 256, 128, 7, 1), (64, 96, 264, 40, 4, 1), (200, 640, 1152, 32, 6, 3), (1030, 512, 768, 64, 3, 2),
    # at most 16 rows: one launch up to 72 K values of an adapter and its rows, two above
    (16, 1024, 1536, 8, 16, 3), (13, 520, 4136, 64, 5, 1), (7, 1000, 72, 40, 2, 1), (2, 4096, 2048, 16, 1, 1), (9, 2000, 1040, 32, 4, 1),
    (3000, 2048, 1024, 16, 20, 1), (129, 4104, 2056, 104, 9, 1), (100, 72, 4096, 128, 3, 4)])
def test_an_adapter_per_row(dev, m, k, n, r, a, parts):
    say("rows", m, k, n, r, a, parts)
    x, down, up, scale, base, index = make(dev, m, k, n, r, a, parts, seed=m)
    check(adapters.low_rank(x, down, up, index, scale=scale, base=base, parts=parts), x, down, up, index, scale, base, parts)


@pytest.mark.parametrize("b,s,k,n,r,parts", [(3, 1, 128, 128, 16, 1), (5, 3, 1024, 640, 24, 1), (1, 16, 512, 192, 8, 3), (2, 77, 320, 384, 8, 3), (5, 16, 512, 128, 32, 1),
                                             (2, 1024, 1024, 512, 48, 1)])
def test_an_adapter_per_sequence(dev, b, s, k, n, r, parts):
    say("sequences", b, s, k, n, r, parts)
    x, down, up, scale, base, _ = make(dev, b * s, k, n, r, 4, parts, seed=s)
    index = torch.tensor([3, -1, 0, 2, 3][:b], dtype=torch.int32, device=dev)
    out = adapters.low_rank(x.view(b, s, k), down, up, index, scale=scale, base=base.view(b, s, n), parts=parts)
    assert out.shape == (b, s, n)
    check(out, x, down, up, index.repeat_interleave(s), scale, base, parts)
    if b > 1:                                  # sequence 1 has no adapter: its rows are the base
        assert torch.equal(out[1], base.view(b, s, n)[1])


def test_without_base_and_scale(dev):
    say("no base, no scale")
    x, down, up, _, _, index = make(dev, 70, 256, 136, 16, 3)
    out = adapters.low_rank(x, down, up, index)
    check(out, x, down, up, index)
    assert not out[index < 0].any()


def test_in_place_strided_and_views(dev):
    """out over base; rows of wider buffers; what lies beside them keeps its values."""
    say("in place, strided")
    x, down, up, scale, base, index = make(dev, 90, 256, 136, 24, 3)
    want = adapters.low_rank(x, down, up, index, scale=scale, base=base)
    wide_x = torch.full((90, 300), 9.0, dtype=torch.bfloat16, device=dev)[:, :296]
    wide_x[:, 16:272] = x
    wide = torch.full((90, 160), 5.0, dtype=torch.bfloat16, device=dev)
    wide[:, 8:144] = base
    y = wide[:, 8:144]
    assert wide_x[:, 16:272].stride(0) % 8 == 4    # refused: rows not 16-byte aligned
    from qwen_image_accel import _native
    with pytest.raises(_native.Unsupported):
        adapters.low_rank(wide_x[:, 16:272], down, up, index, scale=scale, base=y, out=y)
    wide_x = torch.full((90, 304), 9.0, dtype=torch.bfloat16, device=dev)
    wide_x[:, 16:272] = x
    assert adapters.low_rank(wide_x[:, 16:272], down, up, index, scale=scale, base=y, out=y) is y
    assert torch.equal(y, want)
    assert (wide[:, :8] == 5).all() and (wide[:, 144:] == 5).all()


@pytest.mark.parametrize("m", [9, 90])
def test_out_beside_x_and_over_other_rows(dev, m):
    """x, base and out as columns of one buffer; rows of out that are others' rows of x or base are refused."""
    say("shared buffer", m)
    x, down, up, scale, base, index = make(dev, m, 128, 128, 8, 3)
    want = adapters.low_rank(x, down, up, index, scale=scale, base=base)
    buf = torch.cat([x, base, torch.zeros_like(base)], 1)
    bx, bb, bo = buf[:, :128], buf[:, 128:256], buf[:, 256:]
    assert torch.equal(adapters.low_rank(bx, down, up, index, scale=scale, base=bb, out=bo), want)
    assert torch.equal(bx, x) and torch.equal(bb, base)
    tall = torch.zeros(m + 1, 128, dtype=torch.bfloat16, device=dev)
    for kw in (dict(x=x, base=base, out=x), dict(x=x, base=tall[1:], out=tall[:-1]), dict(x=tall[:-1], base=base, out=tall[1:]),
               dict(x=bx, base=bb, out=buf[:, 64:192])):
        with pytest.raises(_native.QimError, match="overlaps"):
            adapters.low_rank(kw["x"], down, up, index, scale=scale, base=kw["base"], out=kw["out"])
    with pytest.raises(_native.Unsupported):
        adapters.low_rank(x[:, :0], down[:, :, :0].contiguous(), up, index, base=base)


def test_entries_outside_the_adapters_mean_none(dev):
    say("index outside")
    x, down, up, scale, base, index = make(dev, 40, 128, 128, 8, 3)
    index[::2] = torch.tensor([3, 1000, -5, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=dev).repeat(4)
    out = adapters.low_rank(x, down, up, index, scale=scale, base=base)
    assert torch.equal(out[::2], base[::2])
    check(out, x, down, up, torch.where((index < 0) | (index > 2), -1, index), scale, base)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_request_keeps_its_values_to_itself(dev, value):
    """NaN or infinities in one adapter, or in one row of x, reach that adapter's rows, or that row, only."""
    say("isolation", value)
    x, down, up, scale, base, index = make(dev, 50, 256, 128, 16, 4)
    want = adapters.low_rank(x, down, up, index, scale=scale, base=base)
    for t in (down, up, scale):
        keep = t.clone()
        t[2] = value
        out = adapters.low_rank(x, down, up, index, scale=scale, base=base)
        assert torch.equal(out[index != 2], want[index != 2])
        assert not out[index == 2].isfinite().any()
        t.copy_(keep)
    row = int((index == 1).nonzero()[0])
    x[row, 3] = value
    out = adapters.low_rank(x, down, up, index, scale=scale, base=base)
    rest = torch.arange(50, device=dev) != row
    assert torch.equal(out[rest], want[rest]) and not out[row].isfinite().any()


def test_result_does_not_depend_on_the_neighbours(dev):
    """A row gives the same bits whichever rows are beside it (same number of rows: the same split over K)."""
    say("neighbours")
    x, down, up, scale, base, index = make(dev, 64, 512, 256, 16, 5)
    want = adapters.low_rank(x, down, up, index, scale=scale, base=base)
    perm = torch.randperm(64, generator=torch.Generator().manual_seed(0)).to(dev)
    out = adapters.low_rank(x[perm].contiguous(), down, up, index[perm].contiguous(), scale=scale, base=base[perm].contiguous())
    assert torch.equal(out, want[perm])


def test_nothing(dev):
    say("no rows")
    x, down, up, scale, base, index = make(dev, 8, 64, 64, 8, 2)
    assert adapters.low_rank(x[:0], down, up, index[:0], scale=scale, base=base[:0]).shape == (0, 64)


def test_offsets_past_32_bits(dev):
    """A batch whose output has more than 2^32 elements' bytes: the last rows."""
    m, k, n, r = 190000, 32, 12288, 8
    say("low rank > 2^31 elements", m * n)
    g = torch.Generator().manual_seed(2)
    x, down, up = bf16_randn(g, (m, k)).to(dev), bf16_randn(g, (2, r, k)).to(dev), bf16_randn(g, (2, n, r)).to(dev)
    index = torch.zeros(m, dtype=torch.int32, device=dev)
    index[-5:] = 1
    base = torch.ones(m, n, dtype=torch.bfloat16, device=dev)
    out = adapters.low_rank(x, down, up, index, base=base, out=base)
    for rows in (slice(0, 40), slice(m - 40, m)):
        check(out[rows], x[rows], down, up, index[rows], None, torch.ones(40, n, dtype=torch.bfloat16, device=dev))
