"""Packing and quantizing of 4-bit weights (no GPU needed)."""
import pytest
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import fourbit


def raw(n, k, group, zeros, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scales = torch.rand(n, k // group, generator=g).to(torch.bfloat16)
    return codes, scales, torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None


@pytest.mark.parametrize("n,k,group,zeros", [(1, 32, 32, False), (16, 128, 128, True), (17, 192, 64, True), (40, 416, 32, True)])
def test_packing_keeps_every_code(n, k, group, zeros):
    codes, scales, z = raw(n, k, group, zeros)
    w = fourbit.pack_weight(codes, scales, zeros=z)
    assert (w.rows, w.width, w.group, w.kind) == (n, k, group, "int4")
    assert w.codes.shape == ((n + 15) // 16, (k + 127) // 128, 64, 16)
    back = fourbit.unpack_weight(w)
    assert torch.equal(back[0], codes) and torch.equal(back[1], scales) and (z is None or torch.equal(back[2], z))
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(1).float().unflatten(1, (-1, group))
    want = (q - (8.0 if z is None else z.float().unsqueeze(-1))) * scales.float().unsqueeze(-1)
    assert torch.equal(fourbit.dequantize_weight(w), want.flatten(1))


def test_where_a_code_lies():
    """Row 19, k = 128 + 32 * 2 + 8 * 3 + e: tile 1, step 1, lane 3 + 16 * 3, dword 2."""
    for kind, places in (("int4", [(e % 4, 4 * (e // 4)) for e in range(8)]), ("mxfp4", [(e // 2, 4 * (e % 2)) for e in range(8)])):
        for e, (byte, shift) in enumerate(places):
            k = 128 + 64 + 24 + e
            codes = torch.zeros(20, 128, dtype=torch.uint8)
            codes[19, k // 2] = 13 << (4 * (k % 2))
            scales = torch.ones(20, 8, dtype=torch.bfloat16) if kind == "int4" else torch.full((20, 8), 127, dtype=torch.uint8)
            w = fourbit.pack_weight(codes, scales)
            want = torch.zeros_like(w.codes)
            want[1, 1, 3 + 16 * 3, 4 * 2 + byte] = 13 << shift
            assert torch.equal(w.codes, want)


def test_mxfp4_exponents_by_step():
    codes = torch.zeros(3, 96, dtype=torch.uint8)
    scales = torch.arange(18, dtype=torch.uint8).view(3, 6)
    w = fourbit.pack_weight(codes, scales.view(torch.float8_e8m0fnu))
    assert w.kind == "mxfp4" and w.scales.shape == (1, 2, 16, 4)
    assert w.scales[0, 0, 2].tolist() == [12, 13, 14, 15] and w.scales[0, 1, 2].tolist() == [16, 17, 0, 0]
    assert torch.equal(fourbit.unpack_weight(w)[1], scales)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_int4_is_the_nearest_code(group):
    w = torch.randn(9, 256, generator=torch.Generator().manual_seed(1))
    w[3] = 0
    w[4] = w[4].abs() + 1
    for symmetric in (False, True):
        q = fourbit.quantize_weight(w, "int4", group, symmetric=symmetric)
        _, scales, zeros = fourbit.unpack_weight(q)
        assert (zeros is None) == symmetric
        s = scales.float().repeat_interleave(group, 1)
        err = (fourbit.dequantize_weight(q) - w).abs()
        # half a step; the group's ends may lie past the last code by the zero point's and the scale's roundings:
        # 1/2 and 15 steps times 2^-8
        assert (err <= s * (0.5 + 0.5 + 16 * 2.0 ** -8) + 1e-7).all()
        inner = err <= s * 0.5 * (1 + 1e-6) + 1e-7
        assert inner.float().mean() > 0.9
        assert not fourbit.dequantize_weight(q)[3].any()


def test_mxfp4_is_the_nearest_code_of_the_better_exponent():
    w = torch.randn(8, 128, generator=torch.Generator().manual_seed(2)) * torch.logspace(-3, 3, 8)[:, None]
    w[5, :32] = 0
    q = fourbit.quantize_weight(w, "mxfp4")
    _, e, _ = fourbit.unpack_weight(q)
    table = torch.tensor(fourbit.E2M1 + tuple(-v for v in fourbit.E2M1)).double()
    best = None
    for d in (-1, 0, 1):
        unit = torch.exp2(e.double() + d - 127).repeat_interleave(32, 1).unsqueeze(-1)
        near = (table * unit - w.double().unsqueeze(-1)).abs().amin(-1)
        err = near.square().unflatten(1, (-1, 32)).sum(-1)
        if d == 0:
            got = (fourbit.dequantize_weight(q).double() - w.double()).abs()
            assert torch.allclose(got, near, rtol=1e-6, atol=0)
            mine = err
        best = err if best is None else torch.minimum(best, err)
    assert (mine <= best * (1 + 1e-6) + 1e-30).all()


def test_refusals():
    codes, scales, z = raw(8, 128, 64, True)
    for args, kw in (((codes.int(), scales), {}), ((codes, scales.float()), {}), ((codes, scales[:4]), {}), ((codes[0], scales[0]), {}),
                     ((codes, torch.ones(8, 8, dtype=torch.bfloat16)), {}), ((codes, torch.ones(8, 2, dtype=torch.uint8)), {}),
                     ((codes, scales), dict(zeros=z[:, :1])), ((codes, scales), dict(zeros=z + 16)), ((codes, scales), dict(zeros=z.float())),
                     ((codes, torch.full((8, 4), 255, dtype=torch.uint8)), {}), ((codes[:0], scales[:0]), {})):
        with pytest.raises(ValueError):
            fourbit.pack_weight(*args, **kw)
    w = torch.ones(8, 96)
    for args in ((w, "int4", 64), (w, "int4", 48), (w, "nf4"), (w[0], "mxfp4"), (w[:, :40], "mxfp4"), (w * float("inf"), "mxfp4")):
        with pytest.raises(ValueError):
            fourbit.quantize_weight(*args)


def test_a_weight_put_together_by_hand_is_checked():
    """Sizes that do not belong to the tensors are refused before any address reaches a kernel."""
    mx = fourbit.quantize_weight(torch.randn(20, 256), "mxfp4")
    w = fourbit.quantize_weight(torch.randn(20, 256), "int4", 64)
    cpu = mx.codes.device
    fourbit._check_weight("test", mx, cpu), fourbit._check_weight("test", w, cpu)
    wrong = [mx._replace(group=64), mx._replace(group=64, scales=mx.scales[..., :2].contiguous()), mx._replace(width=384), mx._replace(rows=33),
             mx._replace(zeros=mx.scales), mx._replace(codes=mx.codes.transpose(0, 1)), w._replace(group=32), w._replace(group=48),
             w._replace(rows=0), w._replace(scales=w.scales.view(torch.int16)), w._replace(zeros=w.zeros[..., :1])]
    for bad in wrong:
        with pytest.raises(_native.Unsupported):
            fourbit._check_weight("test", bad, cpu)


def test_a_group_whose_span_passes_fp32():
    g = torch.zeros(16, 64)
    g[:, 0], g[:, 1] = 3e38, -3e38
    back = fourbit.dequantize_weight(fourbit.quantize_weight(g, "int4", 64))
    assert back.isfinite().all() and (back - g).abs().max() <= 2.1e37   # half a step of 4e37 and the scale's own rounding, 2^-9 of 15 / 2 steps
