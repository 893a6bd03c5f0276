"""Refusals of the few-token operators (no GPU): the C entry points reject bad arguments before any launch, the
wrappers host tensors."""
import types

import pytest
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import attention, elementwise, fourbit, kv_cache

ARG, SHAPE, LAYOUT = _native.QIM_ERR_ARG, _native.QIM_ERR_SHAPE, _native.QIM_ERR_LAYOUT
FAR = 1 << 30


def norm(h=FAR, ldh=256, x=2 * FAR, ldx=256, post=0, post_w=None, post_eps=1e-6, gate=16, gate_b=256, alpha=1.0, norm=2, norm_w=None,
         eps=1e-6, scale=16, scale_b=256, shift=None, flags=0, ho=3 * FAR, ldho=256, z=4 * FAR, ldz=256, zs=None, m=8, d=256, seq=4):
    return ("qim_residual_norm", (h, ldh, x, ldx, post, post_w, post_eps, gate, gate_b, alpha, norm, norm_w, eps, scale, scale_b, shift, 0,
                                  flags, ho, ldho, z, ldz, zs, m, d, seq, None))


def four(x=FAR, ldx=256, group=64, codes=16, scales=16, zeros=None, codes2=None, scales2=None, zeros2=None, bias=None, out=2 * FAR,
         ldo=100, f32=0, m=4, n=100, k=256):
    return ("qim_fourbit_matmul", (x, ldx, group, codes, scales, zeros, codes2, scales2, zeros2, bias, out, ldo, f32, m, n, k, None))


def share(q=FAR, ldq=512, pk=16, plens=16, which=16, kc=16, lengths=16, tree=None, o=2 * FAR, ws=16, nbytes=1 << 40, b=2, s=1, p=3, cp=64,
          c=32, h=4, hk=2, d=128, scale=0.1):
    return ("qim_attention_shared", (q, 512, ldq, pk, 16, 16, 16, plens, which, kc, 16, 16, 16, lengths, tree, 0, o, ws, nbytes, b, s, p, cp, c,
                                     h, hk, d, scale, None))


@pytest.mark.parametrize("call,code", [
    (share(q=None), ARG), (share(pk=None), ARG), (share(kc=None), ARG), (share(lengths=None), ARG), (share(o=None), ARG), (share(ws=None), ARG),
    (share(scale=0.0), ARG), (share(scale=float("nan")), ARG), (share(scale=1e31), ARG), (share(nbytes=64), ARG), (share(o=FAR + 512), ARG),
    (share(which=None), SHAPE), (share(p=0), SHAPE), (share(p=4097), SHAPE), (share(cp=0), SHAPE), (share(c=-1), SHAPE), (share(s=65), SHAPE),
    (share(s=0), SHAPE), (share(b=0), SHAPE), (share(h=3), SHAPE), (share(d=64), SHAPE), (share(cp=1 << 31), SHAPE), (share(b=1 << 20), SHAPE),
    (share(h=1 << 17, hk=1), SHAPE), (share(b=1 << 19, s=64, p=1), SHAPE), (share(cp=1 << 30, p=4096), SHAPE),
    (share(q=FAR + 8), LAYOUT), (share(ldq=500), LAYOUT), (share(ldq=256), LAYOUT), (share(pk=24), LAYOUT), (share(o=2 * FAR + 8), LAYOUT),
    (share(ws=24), LAYOUT), (share(lengths=18), LAYOUT), (share(which=18), LAYOUT), (share(plens=17), LAYOUT),
    (norm(h=None), ARG), (norm(x=None), ARG), (norm(ho=None), ARG), (norm(z=None), ARG), (norm(post=3), ARG), (norm(norm=0), ARG),
    (norm(norm=3), ARG), (norm(flags=8), ARG), (norm(post_w=16), ARG), (norm(norm_w=16), ARG), (norm(scale=None, flags=1), ARG),
    (norm(flags=4, gate=None), ARG), (norm(flags=4, scale=None), ARG), (norm(flags=4, alpha=0.5), ARG), (norm(flags=4, norm=1), ARG),
    (norm(flags=4, post=1), ARG), (norm(alpha=float("nan")), ARG), (norm(alpha=float("inf")), ARG), (norm(eps=-1.0), ARG),
    (norm(eps=float("nan")), ARG), (norm(post=1, post_eps=-1.0), ARG),
    (norm(m=0), SHAPE), (norm(d=0), SHAPE), (norm(d=252), SHAPE), (norm(d=16392, ldh=16392), SHAPE), (norm(zs=16, d=248), SHAPE),
    (norm(seq=0), SHAPE), (norm(m=1 << 22), SHAPE), (norm(m=(1 << 22) - 1, zs=16), SHAPE), (norm(seq=1 << 31), SHAPE),
    (norm(ldh=248), LAYOUT), (norm(ldx=260), LAYOUT), (norm(ldho=8), LAYOUT), (norm(ldz=100), LAYOUT), (norm(gate_b=100), LAYOUT),
    (norm(scale_b=-8), LAYOUT), (norm(h=FAR + 8), LAYOUT), (norm(gate=8), LAYOUT), (norm(zs=8), LAYOUT),
    # outputs over inputs at another place or stride, over each other, and codes over rows
    (norm(ho=FAR + 16), ARG), (norm(ho=FAR, ldho=264), ARG), (norm(ho=2 * FAR - 16), ARG), (norm(z=FAR + 512), ARG),
    (norm(z=3 * FAR), ARG), (norm(zs=16, z=FAR), ARG), (norm(zs=2 * FAR, z=16), ARG), (norm(zs=16, z=3 * FAR - 128 * 256 + 16), ARG),
    (four(x=None), ARG), (four(codes=None), ARG), (four(scales=None), ARG), (four(out=None), ARG), (four(codes2=16), ARG),
    (four(scales2=16), ARG), (four(group=16), ARG), (four(group=0, zeros=16), ARG), (four(zeros2=16), ARG),
    (four(codes2=16, scales2=16, zeros=16), ARG), (four(codes2=16, scales2=16, bias=16), ARG), (four(f32=2), ARG),
    (four(m=0), SHAPE), (four(n=0), SHAPE), (four(k=0), SHAPE), (four(k=224), SHAPE), (four(group=0, k=48), SHAPE), (four(m=1 << 20), SHAPE),
    (four(n=1 << 24, ldo=1 << 24), SHAPE), (four(ldx=248), LAYOUT), (four(ldx=260), LAYOUT), (four(ldo=99), LAYOUT), (four(x=FAR + 8), LAYOUT),
    (four(codes=24), LAYOUT), (four(scales=8), LAYOUT), (four(zeros=8), LAYOUT), (four(out=2 * FAR + 1), LAYOUT),
    (four(out=2 * FAR + 2, f32=1), LAYOUT), (four(bias=17), LAYOUT), (four(out=FAR + 2 * 256), ARG), (four(out=FAR - 8 * 99), ARG)])
def test_entry_points_refuse(call, code):
    name, args = call
    rc = getattr(_native.lib(), name)(*args)
    assert rc == code, (rc, _native.lib().qim_last_error())
    assert _native.lib().qim_last_error()


def test_workspace_sizes():
    size = _native.lib().qim_attention_shared_workspace_bytes
    assert size(2, 1, 64, 32, 4, 2, 1, 0) > 0 and size(2, 1, 64, 0, 4, 2, 1, 0) > 0      # an own cache of no positions
    assert size(2, 65, 64, 32, 4, 2, 1, 0) == 0 and size(2, 1, 64, 32, 4, 2, 2, 0) == 0  # not shapes it takes
    assert size(48, 1, 32768, 640, 32, 8, 5, 1) >= 48 * 32 * 2 * 128 * 4                 # a prefix's and an own result of every row


def test_wrappers_refuse_host_tensors():
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    w = fourbit.quantize_weight(torch.ones(16, 128))
    with pytest.raises(_native.Unsupported):
        fourbit.matmul(x, w)
    with pytest.raises(_native.Unsupported):
        fourbit.swiglu(x, w, w)
    cache = kv_cache.empty_cache(1, 8, 2, 128, "cpu")
    with pytest.raises(_native.Unsupported):
        attention.attention_shared(torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16), cache, cache, torch.ones(1, dtype=torch.int32))
    with pytest.raises(_native.Unsupported):
        elementwise.residual_norm(x, x, types.SimpleNamespace(weight=None, eps=1e-6))
