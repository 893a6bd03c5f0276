"""A launch holds fewer than 2^32 threads along its grid: larger problems of the
many-request operators are refused by their shape, before a launch."""
import pytest

from qwen_image_accel import _native

BIG = 1 << 40


@pytest.mark.parametrize("name,args", [
    # positions of one head: a wave each, for K and for V
    ("qim_cache_read", (16, 16, 16, 16, 16, 16, 1, 1 << 25, 1 << 25, 1, 128, None)),
    ("qim_cache_read", (16, 16, 16, 16, 16, 16, 1 << 12, 1 << 13, 1 << 13, 1, 64, None)),
    ("qim_cache_write", (16, 1 << 32, 128, 16, 1 << 32, 128, 16, 16, 16, 16, None, 0, None, 1, 1 << 25, 1 << 25, 1, 128, None)),
    # a workgroup of 512 threads per 64 rows, or of 256 per 32 rows and 1024 columns
    ("qim_low_rank", (16, 8, 16, 16, 16, None, None, 0, BIG, 1 << 12, 16, BIG, 1 << 29, 1, 8, 1 << 12, 8, 1, 1, None)),
    ("qim_low_rank", (16, 8, 16, 16, 16, None, None, 0, BIG, 1 << 23, 16, BIG, 1 << 20, 1, 8, 1 << 23, 8, 1, 1, None)),
])
def test_grids_past_32_bits_are_refused(name, args):
    rc = getattr(_native.lib(), name)(*args)
    assert rc == _native.QIM_ERR_SHAPE, (rc, _native.lib().qim_last_error())
    assert b"too large" in _native.lib().qim_last_error()
