"""The residual with the norms on both of its sides against float64 and, in its eager form, against the
operators that it joins."""
import types

import pytest
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import elementwise, epilogue, layernorm, mxfp8
from qwen_image_accel.weights import unswizzle_scales
from tests import few_tokens_ref as R
from tests.helpers import bf16_randn

pytestmark = pytest.mark.gpu


def say(*a):
    print("[case]", *a, flush=True)


def rms(w, eps=1e-6):
    return types.SimpleNamespace(weight=w, bias=None, eps=eps)


def layer(d, eps=1e-6):
    return types.SimpleNamespace(normalized_shape=(d,), elementwise_affine=False, eps=eps)


def plain(norm):
    if norm is None:
        return None
    return ("layer", None, norm.eps) if hasattr(norm, "normalized_shape") else ("rms", norm.weight, norm.eps)


def make(dev, b, s, d, post, norm, mod, seed=0, offset=0.0):
    g = torch.Generator().manual_seed(seed)

    def randn(*shape, scale=1.0):
        return bf16_randn(g, shape, scale).to(dev)

    def of(kind):
        return None if kind == "none" else layer(d) if kind == "layer" else rms((1 + randn(d, scale=0.2)).to(torch.bfloat16))
    h, x = (randn(b, s, d, scale=2.0).float() + offset).to(torch.bfloat16), randn(b, s, d)
    shapes = {"none": (), "each": ((b, 1, d),) * 3, "all": ((d,), (1, 1, d), (d,))}[mod]
    gate, scale, shift = [randn(*v, scale=0.5) for v in shapes] or (None,) * 3
    return h, x, of(norm), dict(post=of(post), gate=gate, scale=scale, shift=shift)


def reference(h, x, norm, post, gate, scale, shift, alpha, add_one):
    return R.residual_norm(h, x, plain(norm), gate, alpha, plain(post), scale, shift, add_one)


def check(h, x, norm, kw, alpha, add_one, got):
    hs, bh, z, ez = reference(h, x, norm, alpha=alpha, add_one=add_one, **kw)
    for name, a, want, bound in (("h", got[0], hs, bh), ("z", got[1], z, R.rounded(z, ez))):
        err = (a.double().cpu() - want).abs()
        assert a.isfinite().all() and (err <= bound).all(), (name, float((err / bound).max()))


@pytest.mark.parametrize("b,s,d", [(1, 1, 8), (3, 1, 72), (2, 5, 512), (1, 3, 1000), (16, 1, 4096), (2, 130, 4096), (1, 2, 8192),
                                   (1, 2, 8200), (2, 3, 16384)])
@pytest.mark.parametrize("post,norm,mod", [("none", "layer", "each"), ("rms", "rms", "none"), ("layer", "rms", "all"),
                                           ("rms", "layer", "each")])
def test_against_float64(dev, b, s, d, post, norm, mod):
    say("residual_norm", b, s, d, post, norm, mod)
    h, x, n, kw = make(dev, b, s, d, post, norm, mod, seed=d + s)
    for alpha, add_one in ((1.0, True), (0.375, False)):
        got = elementwise.residual_norm(h, x, n, residual_scale=alpha, add_one=add_one, **kw)
        check(h, x, n, kw, alpha, add_one and kw["scale"] is not None, got)


def test_a_mean_far_from_zero(dev):
    """Rows whose mean is 256 deviations away: the variance is a small difference of large sums."""
    say("far mean")
    h, x, n, kw = make(dev, 2, 9, 1536, "layer", "layer", "each", seed=5, offset=512.0)
    check(h, x, n, kw, 1.0, True, elementwise.residual_norm(h, x, n, add_one=True, **kw))


def test_rows_that_do_not_fit_fp32_squares(dev):
    """Magnitudes whose squares leave fp32, and rows of zeros."""
    say("magnitudes")
    h, x, n, kw = make(dev, 1, 4, 256, "rms", "rms", "none", seed=6)
    h[:, 1] *= 2.0 ** 100
    h[:, 2] *= 2.0 ** -100
    x[:, 2] *= 2.0 ** 90
    h[:, 3] = 0
    x[:, 3] = 0
    got = elementwise.residual_norm(h, x, n, **kw)
    check(h, x, n, kw, 1.0, False, got)
    assert not got[1][:, 3].any()


def test_a_row_of_nan_stays_alone(dev):
    say("nan row")
    h, x, n, kw = make(dev, 2, 4, 264, "rms", "layer", "each", seed=7)
    want = elementwise.residual_norm(h, x, n, **kw)
    x[0, 2, 5], h[1, 1, 0] = float("nan"), float("inf")
    got = elementwise.residual_norm(h, x, n, **kw)
    hit = torch.zeros(2, 4, dtype=torch.bool, device=dev)
    hit[0, 2] = hit[1, 1] = True
    for a, w in zip(got, want):
        assert torch.equal(a[~hit], w[~hit])
    assert got[0][0, 2].isnan().all() and got[1][0, 2].isnan().all() and not got[1][1, 1].isfinite().any()


def test_strides_and_places(dev):
    """Rows apart, vectors that are rows of one modulation tensor, h' over h and over x, two-dimensional inputs."""
    say("strides")
    b, s, d = 3, 7, 640
    h, x, n, kw = make(dev, b, s, d, "rms", "rms", "each", seed=8)
    want = elementwise.residual_norm(h, x, n, **kw)
    wide = torch.randn(b, s, 2 * d + 8, device=dev).to(torch.bfloat16)
    keep = wide.clone()
    hw, xw = wide[..., :d], wide[..., d:2 * d]
    hw.copy_(h)
    xw.copy_(x)
    mod = torch.stack([kw[k][:, 0] for k in ("gate", "scale", "shift")], 1)           # (b, 3, d)
    kv = dict(post=kw["post"], gate=mod[:, 0:1], scale=mod[:, 1:2], shift=mod[:, 2:3])
    got = elementwise.residual_norm(hw, xw, n, out=xw, **kv)
    assert got[0] is xw and torch.equal(xw, want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(hw, h) and torch.equal(wide[..., 2 * d:], keep[..., 2 * d:])
    h2 = h.clone()
    got = elementwise.residual_norm(h2, x, n, out=h2, **kw)
    assert torch.equal(h2, want[0]) and torch.equal(got[1], want[1])
    one = {k: (v[1:2] if isinstance(v, torch.Tensor) else v) for k, v in kw.items()}
    got = elementwise.residual_norm(h[1], x[1], n, **one)
    assert torch.equal(got[0], want[0][1]) and torch.equal(got[1], want[1][1])
    empty = elementwise.residual_norm(h[:, :0], x[:, :0], n, **kw)
    assert empty[0].shape == empty[1].shape == (b, 0, d)


@pytest.mark.parametrize("tiled", [False, True])
@pytest.mark.parametrize("b,s,d", [(1, 1, 128), (2, 65, 1152), (1, 257, 4096)])
def test_codes(dev, b, s, d, tiled):
    """MXFP8 output: the exponent brings the block's largest value to 224..448, every code is within half an E4M3
    step (2^-4 of the value, 2^-10 of the block's unit) of the value, padding rows are zeros."""
    say("codes", b, s, d, tiled)
    h, x, n, kw = make(dev, b, s, d, "rms", "layer", "each", seed=d)
    got, z = elementwise.residual_norm(h, x, n, add_one=True, quantized=True, tiled=tiled, **kw)
    hs, bh, want, ez = reference(h, x, n, alpha=1.0, add_one=True, **kw)
    assert ((got.double().cpu() - hs).abs() <= bh).all()
    assert z.tiled == tiled and z.rows == b * s and z.shape == h.shape
    rows = mxfp8.as_row_major(z)
    e = unswizzle_scales(rows.scales, b * s, d).cpu().int()
    codes = rows.values.cpu().float()
    assert not codes[b * s:].any() and not e[b * s:].any()
    unit = torch.exp2(e[:b * s].double() - 127).repeat_interleave(32, 1)
    w, tol = want.reshape(-1, d), ez.reshape(-1, d)
    err = (codes[:b * s].double() * unit - w).abs()
    assert (err <= tol + 2.0 ** -4 * (w.abs() + tol) + 2.0 ** -10 * unit).all()
    top = (w / unit).abs().unflatten(1, (-1, 32)).amax(-1)
    slack = (tol / unit).unflatten(1, (-1, 32)).amax(-1)
    assert (top - slack <= 448).all() and (top + slack > 224).all()


@pytest.mark.parametrize("b,s,d", [(1, 1, 128), (2, 37, 640), (3, 64, 1536), (2, 100, 4096), (1, 5, 8192), (1, 3, 16384)])
@pytest.mark.parametrize("shift,add_one", [(False, False), (True, True)])
def test_eager_form_has_the_bits_of_its_parts(dev, b, s, d, shift, add_one):
    say("eager", b, s, d, shift, add_one)
    h, x, n, kw = make(dev, b, s, d, "none", "layer", "each", seed=s)
    norm = torch.nn.LayerNorm(d, eps=1e-6, elementwise_affine=False)
    t = kw["shift"] if shift else None
    want_h = elementwise.residual(h, x, kw["gate"])
    args = dict(gate=kw["gate"], scale=kw["scale"], shift=t, add_one=add_one, rounding="eager")
    got = elementwise.residual_norm(h, x, norm, **args)
    want = layernorm.layer_norm_scale(want_h, kw["scale"], norm, shift=t, add_one=add_one)
    assert torch.equal(got[0], want_h) and torch.equal(got[1], want)
    for tiled in (False, True):
        got = elementwise.residual_norm(h, x, norm, quantized=True, tiled=tiled, **args)
        want = epilogue.layer_norm_scale_quantize(want_h, kw["scale"], norm, shift=t, add_one=add_one, tiled=tiled)
        assert torch.equal(got[0], want_h)
        assert torch.equal(got[1].values.view(torch.uint8), want.values.view(torch.uint8))
        assert torch.equal(got[1].scales.view(torch.uint8), want.scales.view(torch.uint8))


def test_eager_rows_that_need_the_second_pass(dev):
    """A mean far from 0, rows of one value, a row with NaN: the eager form's variance takes its exact path."""
    say("eager second pass")
    h, x, n, kw = make(dev, 1, 16, 1536, "none", "layer", "each", seed=3, offset=512.0)
    h[:, 3], x[:, 3] = 7.0, 0.0
    h[:, 4, 9] = float("nan")
    norm = torch.nn.LayerNorm(1536, eps=1e-6, elementwise_affine=False)
    want_h = elementwise.residual(h, x, kw["gate"])
    want = layernorm.layer_norm_scale(want_h, kw["scale"], norm)
    got = elementwise.residual_norm(h, x, norm, gate=kw["gate"], scale=kw["scale"], rounding="eager")
    assert torch.equal(got[0].view(torch.int16), want_h.view(torch.int16))
    live = torch.arange(16, device=dev) != 4
    assert torch.equal(got[1][:, live], want[:, live]) and got[1][:, 4].isnan().all()


def test_streams_and_graphs(dev):
    say("graph")
    h, x, n, kw = make(dev, 2, 33, 512, "rms", "rms", "each", seed=4)
    out = torch.empty_like(h)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = elementwise.residual_norm(h, x, n, out=out, **kw)
    torch.cuda.current_stream().wait_stream(side)
    want = elementwise.residual_norm(h, x, n, **kw)
    assert torch.equal(first[0], want[0]) and torch.equal(first[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = elementwise.residual_norm(h, x, n, out=out, **kw)
    for i in range(3):
        x.copy_(torch.randn_like(x.float()).to(torch.bfloat16))
        graph.replay()
        want = elementwise.residual_norm(h, x, n, **kw)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i


def test_refusals(dev):
    say("refusals")
    U = _native.Unsupported
    h, x, n, kw = make(dev, 2, 3, 64, "none", "layer", "each")
    rn = elementwise.residual_norm
    for bad in (dict(gate=torch.cat([kw["gate"]] * 2)), dict(gate=kw["gate"].float()), dict(scale=kw["scale"].expand(2, 3, 64)),
                dict(gate=torch.zeros(2, 1, 128, dtype=torch.bfloat16, device=dev)[..., ::2]),
                dict(post=rms(torch.ones(32, dtype=torch.bfloat16, device=dev))), dict(post=rms(torch.ones(64, device=dev))),
                dict(post=torch.nn.LayerNorm(64).to(dev)), dict(post=layer(32)),
                dict(gate=torch.zeros(2 * 68, dtype=torch.bfloat16, device=dev).as_strided((2, 1, 64), (68, 64, 1)))):
        with pytest.raises(U):
            rn(h, x, n, **bad)
    for args in ((h.float(), x, n), (h, x[:, :2], n), (h, x[..., ::2], n), (h[0, 0], x[0, 0], n), (h.cpu(), x, n)):
        with pytest.raises(U):
            rn(*args)
    with pytest.raises(U):
        rn(h, x, n, quantized=True)                        # D a multiple of 128
    for bad in (dict(), dict(gate=kw["gate"]), dict(gate=kw["gate"], scale=kw["scale"], residual_scale=0.5),
                dict(gate=kw["gate"], scale=kw["scale"], post=rms(None))):
        with pytest.raises(_native.QimError):
            rn(h, x, n, rounding="eager", **bad)
    with pytest.raises(ValueError):
        rn(h, x, n, rounding="twice")
    with pytest.raises(ValueError):
        rn(h, x, None)
    wide = torch.zeros(2, 3, 128, dtype=torch.bfloat16, device=dev)
    with pytest.raises(_native.QimError):
        rn(wide[..., :64], x, n, out=wide[..., 8:72])
    with pytest.raises(U):
        rn(h, x, n, out=torch.empty_like(h).float())
