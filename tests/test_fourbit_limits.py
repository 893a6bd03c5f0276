"""The largest problems of the 4-bit products: refused by their shape before any launch (no GPU)."""
import pytest
import torch

from qwen_image_accel import _native
from tests.test_few_tokens_refusals import FAR, SHAPE, four

M = (1 << 20) - 1


def code(call):
    return getattr(_native.lib(), call[0])(*call[1])


@pytest.mark.parametrize("call", [
    four(m=M, n=1 << 20, ldo=1 << 20), four(m=M, n=(1 << 24) - 1, ldo=1 << 24, out=64 * FAR), four(m=M, n=1 << 20, ldo=1 << 20, group=0),
    four(m=M, n=1 << 17, ldo=1 << 17, group=32), four(m=M, n=21000, ldo=21000, codes2=16, scales2=16),
    four(m=M, n=21000, ldo=21000, codes2=16, scales2=16, group=128),
    four(m=M, n=(1 << 24) - 1, ldo=1 << 24, out=64 * FAR, codes2=16, scales2=16, group=0)])   # (the workgroups' number wraps in 32 bits)
def test_more_than_2_32_threads(call):
    assert code(call) == SHAPE, _native.lib().qim_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="an accepted call launches, and its addresses are made up")
def test_large_problems_below_that_are_taken():
    for call in (four(m=M, n=16000, ldo=16000, codes2=16, scales2=16), four(m=M, n=35000, ldo=35000), four(m=M, n=40000, ldo=40000, group=0)):
        assert code(call) == _native.QIM_ERR_LAUNCH
