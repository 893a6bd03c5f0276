"""Where rows of the MXFP8 K/V cache may be written and read: positions past what the
arguments' types hold, and caches of no positions."""
import pytest
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import kv_cache
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
