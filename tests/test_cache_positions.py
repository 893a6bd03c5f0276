"""Where rows of the MXFP8 K/V cache may be written and read: positions past what the
arguments' types hold, caches of no positions, and prefixes of any strides."""
import pytest
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import attention, kv_cache
from qwen_image_accel.optimizations.prefix_cache import QuantizedLayerCache
from tests.helpers import bf16_randn


def say(*a):
    print("[case]", *a, flush=True)


@pytest.mark.parametrize("first", [9, 2 ** 31, 2 ** 62, 2 ** 63 - 8, 2 ** 63 - 1, -2 ** 63])
def test_a_first_position_past_the_cache_is_refused(first):
    """first + S does not wrap around."""
    rc = _native.lib().qim_cache_write(16, 4096, 512, 16, 4096, 512, 16, 16, 16, 16, None, first, None, 2, 8, 16, 4, 128, None)
    assert rc == _native.QIM_ERR_ARG, (rc, _native.lib().qim_last_error())


@pytest.mark.gpu
@pytest.mark.parametrize("start", [7, 2 ** 63 - 1, 2 ** 64, 2 ** 64 + 3, -2 ** 64, -1])
def test_a_start_that_no_64_bits_hold_is_refused(dev, start):
    say("start", start)
    cache = kv_cache.empty_cache(2, 8, 2, 128, dev)
    for t in cache:
        t.view(torch.uint8).fill_(0x38)
    x = bf16_randn(torch.Generator().manual_seed(0), (2, 2, 2, 128)).to(dev)
    with pytest.raises(_native.QimError):
        kv_cache.write_cache(cache, x, x, start=start)
    torch.cuda.synchronize()
    assert all(bool((t.view(torch.uint8) == 0x38).all()) for t in cache)


@pytest.mark.gpu
def test_a_cache_of_no_positions(dev):
    """No key to see, nowhere to write, nothing to read: zeros, nothing, empty; a host start does not fit."""
    say("no positions")
    cache = kv_cache.empty_cache(2, 0, 2, 128, dev)
    x = bf16_randn(torch.Generator().manual_seed(0), (2, 3, 2, 128)).to(dev)
    n = torch.tensor([5, 0], dtype=torch.int32, device=dev)
    kv_cache.write_cache(cache, x, x, start=n)
    with pytest.raises(_native.QimError):
        kv_cache.write_cache(cache, x, x, start=0)
    assert [t.shape for t in kv_cache.read_cache(cache)] == [(2, 0, 2, 128)] * 2
    tree = torch.ones(3, 3, dtype=torch.bool, device=dev)
    out = torch.full_like(x, 7.0)
    assert attention.attention_cached(x, cache, n, tree=tree, out=out) is out and not out.any()
    assert not attention.attention_cached(x[:, :1], cache, n).any()
    with pytest.raises(_native.Unsupported):
        attention.attention_cached(torch.zeros(2, 65, 2, 128, dtype=torch.bfloat16, device=dev), cache, n)
    with pytest.raises(_native.Unsupported):
        attention.attention_cached(torch.zeros(2, 1, 3, 128, dtype=torch.bfloat16, device=dev), cache, n)


@pytest.mark.gpu
def test_a_prefix_of_any_strides_becomes_a_quantized_layer_cache(dev):
    """Views whose heads are not packed, whose rows are not 16-byte aligned, or of one prompt for several sequences."""
    say("strided prefixes")
    g = torch.Generator().manual_seed(0)
    wide = bf16_randn(g, (2, 4, 9, 132)).to(dev)          # (B, H, P, ...)
    views = [wide[..., :128].transpose(1, 2), wide[..., 4:].transpose(1, 2), wide[:, :, :, :128].transpose(1, 2)[:, 2:7],
             wide[:1, ..., :128].transpose(1, 2).expand(2, 9, 4, 128), bf16_randn(g, (2, 9, 516)).to(dev)[..., 4:].view(2, 9, 4, 128)]
    for view in views:
        got = QuantizedLayerCache(view, view * 2).quantized
        want = QuantizedLayerCache(view.contiguous(), (view * 2).contiguous()).quantized
        for a, b in zip(got, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
