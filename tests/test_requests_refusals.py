"""Refusals of the many-request operators (no GPU): the C entry points reject bad
arguments before any launch, and the Python wrappers tensors they cannot take."""
import ctypes

import pytest
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import adapters, attention, kv_cache

ARG, SHAPE, LAYOUT = _native.QIM_ERR_ARG, _native.QIM_ERR_SHAPE, _native.QIM_ERR_LAYOUT


def write(k=16, ldkb=4096, ldk=512, v=16, kc=16, ks=16, start=None, first=0, count=None, b=2, s=8, c=16, h=4, d=128):
    return ("qim_cache_write", (k, ldkb, ldk, v, 4096, 512, kc, ks, 16, 16, start, first, count, b, s, c, h, d, None))


def read(kc=16, ok=16, b=2, c=16, rows=8, h=4, d=128):
    return ("qim_cache_read", (kc, 16, 16, 16, ok, 16, b, c, rows, h, d, None))


def pack(v=16, kc=16, c=16, p=8, d=128, ldt=512):
    return ("qim_qk_norm_rope_pack_cached", (16, 16, v, kc, 16, 16, 16, c, 16, 16, 16, 16, 16, 16, 1, 4, p, 4, d, ldt, 1e-6,
                                             1e-6, None))


def attend(q=16, ldq=512, kc=16, lengths=16, tree=None, o=16, ws=16, nbytes=1 << 40, b=2, s=1, c=64, h=4, hk=2, d=128,
           scale=0.1):
    return ("qim_attention_cached", (q, 512, ldq, kc, 16, 16, 16, lengths, tree, 0, o, ws, nbytes, b, s, c, h, hk, d, scale, None))


def adapt(x=16, ldx=256, down=16, index=16, base=16, ldb=512, out=16, ldo=512, ws=16, nbytes=1 << 40, m=4, seq=1, k=256, n=512,
          r=16, parts=1, a=2):
    return ("qim_low_rank", (x, ldx, down, 16, index, None, base, ldb, out, ldo, ws, nbytes, m, seq, k, n, r, parts, a, None))


@pytest.mark.parametrize("call,code", [
    (write(k=None), ARG), (write(kc=None), ARG), (write(first=9), ARG), (write(first=-1), ARG), (write(b=0), SHAPE),
    (write(s=0), SHAPE), (write(d=48), SHAPE), (write(ldk=256), LAYOUT), (write(ldk=516), LAYOUT), (write(ldkb=4100), LAYOUT),
    (write(k=24), LAYOUT), (write(ks=8), LAYOUT), (write(b=1 << 20, s=1 << 20, c=1 << 20), SHAPE),
    (read(ok=None), ARG), (read(rows=17), ARG), (read(rows=0), SHAPE), (read(kc=8), LAYOUT), (read(ok=24), LAYOUT),
    (read(d=100), SHAPE), (read(b=1 << 20, c=1 << 20, rows=1 << 20), SHAPE),
    (pack(v=None), ARG), (pack(kc=None), ARG), (pack(p=17), ARG), (pack(kc=24), LAYOUT), (pack(d=96), SHAPE),
    (pack(ldt=256), LAYOUT), (pack(p=-1), SHAPE),
    (attend(q=None), ARG), (attend(lengths=None), ARG), (attend(scale=0.0), ARG), (attend(scale=float("nan")), ARG),
    (attend(ws=None, c=1 << 20), ARG), (attend(nbytes=16, c=1 << 20), ARG), (attend(d=64), SHAPE), (attend(s=65), SHAPE),
    (attend(s=0), SHAPE), (attend(h=3), SHAPE), (attend(c=0), SHAPE), (attend(q=8), LAYOUT), (attend(ldq=500), LAYOUT),
    (attend(o=8), LAYOUT), (attend(lengths=18), LAYOUT), (attend(ws=8, c=1 << 20), LAYOUT),
    (adapt(x=None), ARG), (adapt(index=None), ARG), (adapt(ws=None, m=40), ARG), (adapt(nbytes=15, m=40), ARG), (adapt(m=0), SHAPE),
    (adapt(seq=0), SHAPE), (adapt(k=260), SHAPE), (adapt(r=12), SHAPE), (adapt(r=136), SHAPE), (adapt(parts=3), SHAPE),
    (adapt(n=516), SHAPE), (adapt(ldx=128), LAYOUT), (adapt(ldb=500), LAYOUT), (adapt(ldo=516), LAYOUT), (adapt(x=8), LAYOUT),
    (adapt(down=24), LAYOUT), (adapt(out=8), LAYOUT), (adapt(index=18), LAYOUT),
    # out over x, over base's rows at another place or stride, and over q
    (adapt(out=1 << 20, base=1 << 20, x=(1 << 20) + 1024), ARG), (adapt(out=1 << 20, base=(1 << 20) + 1024), ARG),
    (adapt(out=1 << 20, base=1 << 20, ldb=520), ARG), (adapt(out=1 << 20, ldo=1024, base=(1 << 20) + 1008, ldb=1024), ARG),
    (attend(o=528), ARG), (attend(q=528, o=16), ARG)])
def test_entry_points_refuse(call, code):
    name, args = call
    rc = getattr(_native.lib(), name)(*args)
    assert rc == code, (rc, _native.lib().qim_last_error())
    assert _native.lib().qim_last_error()


def test_workspace_sizes():
    lib = _native.lib()
    assert lib.qim_attention_cached_workspace_bytes(1, 1, 32, 4, 4) == 0          # nothing to split
    assert lib.qim_attention_cached_workspace_bytes(1, 1, 100000, 4, 4) > 0
    assert lib.qim_attention_cached_workspace_bytes(1, 65, 100000, 4, 4) == 0     # not a shape it takes
    assert lib.qim_low_rank_workspace_bytes(400, 1, 256, 16, 3) >= 400 * 48 * 4
    assert lib.qim_low_rank_workspace_bytes(4, 1, 256, 16, 1) == 0                # one launch
    assert lib.qim_low_rank_workspace_bytes(0, 1, 256, 16, 1) == 0


def cpu_cache(b=1, c=8, h=2, d=128):
    return kv_cache.empty_cache(b, c, h, d, "cpu")


def test_wrappers_refuse_host_tensors():
    x = torch.zeros(1, 2, 2, 128, dtype=torch.bfloat16)
    n = torch.ones(1, dtype=torch.int32)
    with pytest.raises(_native.Unsupported):
        kv_cache.write_cache(cpu_cache(), x, x)
    with pytest.raises(_native.Unsupported):
        kv_cache.read_cache(cpu_cache())
    with pytest.raises(_native.Unsupported):
        attention.attention_cached(x, cpu_cache(), n)
    with pytest.raises(_native.Unsupported):
        adapters.low_rank(x[0, 0], x[0], x[0], n)
    with pytest.raises(ValueError, match="multiple of 32"):
        kv_cache.empty_cache(1, 4, 2, 72, "cpu")


@pytest.mark.gpu
def test_wrappers_refuse(dev):
    print("[case] wrapper refusals", flush=True)
    bf, U = torch.bfloat16, _native.Unsupported
    cache = kv_cache.empty_cache(2, 8, 2, 128, dev)
    x = torch.zeros(2, 3, 2, 128, dtype=bf, device=dev)
    n = torch.ones(2, dtype=torch.int32, device=dev)
    for bad in (x.float(), x.cpu(), x[:1], x[..., :64], x.transpose(2, 3).contiguous().transpose(2, 3)):
        with pytest.raises(U):
            kv_cache.write_cache(cache, bad, bad)
        with pytest.raises(U):
            attention.attention_cached(bad, cache, n)
    with pytest.raises(U):
        kv_cache.write_cache(cache, x, x[:, :2])
    for bad in (n.long(), n.cpu(), n[:1], torch.ones(4, dtype=torch.int32, device=dev)[::2]):
        with pytest.raises(U):
            kv_cache.write_cache(cache, x, x, start=bad)
        with pytest.raises(U):
            kv_cache.write_cache(cache, x, x, count=bad)
        with pytest.raises(U):
            attention.attention_cached(x, cache, bad)
    with pytest.raises(_native.QimError):
        kv_cache.write_cache(cache, x, x, start=6)
    for rows in (-1, 9):
        with pytest.raises(ValueError):
            kv_cache.read_cache(cache, rows)
    with pytest.raises(U):
        kv_cache.read_cache(cache._replace(k_exponent=cache.k_exponent[..., :2].contiguous()))
    with pytest.raises(U):
        kv_cache.read_cache(cache._replace(v=cache.v[:, ::2]))
    tree = torch.ones(3, 3, dtype=torch.bool, device=dev)
    for bad in (tree.int(), tree.cpu(), tree[:2], torch.ones(3, 3, 3, dtype=torch.bool, device=dev), torch.ones(3, 6, dtype=torch.bool, device=dev)[:, ::2]):
        with pytest.raises(U):
            attention.attention_cached(x, cache, n, tree=bad)
    with pytest.raises(U):
        attention.attention_cached(torch.zeros(2, 65, 2, 128, dtype=bf, device=dev), cache, n)
    with pytest.raises(U):
        attention.attention_cached(torch.zeros(2, 1, 3, 128, dtype=bf, device=dev), cache, n)
    with pytest.raises(ValueError):
        attention.attention_cached(x, cache, n, out=x[:, :2])
    xr, down, up = torch.zeros(6, 64, dtype=bf, device=dev), torch.zeros(2, 8, 64, dtype=bf, device=dev), torch.zeros(2, 32, 8, dtype=bf, device=dev)
    index, scale = torch.zeros(6, dtype=torch.int32, device=dev), torch.ones(2, device=dev)
    good = dict(x=xr, down=down, up=up, index=index)
    adapters.low_rank(**good, scale=scale)
    for key, bad in (("x", xr.float()), ("x", xr.t().contiguous().t()), ("x", xr[:, :56]), ("down", down.float()), ("down", down[:1]),
                     ("up", up[:, :, :4]), ("up", up.cpu()), ("index", index.long()), ("index", index[:5]), ("index", index.cpu())):
        with pytest.raises(U):
            adapters.low_rank(**{**good, key: bad}, scale=scale)
    for bad in (scale.half(), scale[:1], scale.cpu()):
        with pytest.raises(U):
            adapters.low_rank(**good, scale=bad)
    for key in ("base", "out"):
        for bad in (torch.zeros(6, 31, dtype=bf, device=dev), torch.zeros(6, 32, device=dev), torch.zeros(32, 6, dtype=bf, device=dev).t()):
            with pytest.raises(U):
                adapters.low_rank(**good, **{key: bad})
    with pytest.raises(U):
        adapters.low_rank(**good, parts=2)
