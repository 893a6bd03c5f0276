"""The largest problems of the 4-bit products: refused by their shape before any launch (no GPU); rows far apart (GPU)."""
import pytest
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import fourbit
from qwen_image_accel.optimizations.fourbit import FourBitLinear
from tests.helpers import bf16_randn
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


@pytest.mark.gpu
def test_a_token_of_each_of_some_long_sequences(dev):
    """Rows 2^24 elements apart and more."""
    print("[case] rows far apart", flush=True)
    g = torch.Generator().manual_seed(1)
    w = fourbit.quantize_weight(bf16_randn(g, (40, 4096)).to(dev))
    linear = FourBitLinear.from_packed(w)
    hidden = torch.zeros(5, 4099, 4096, dtype=torch.bfloat16, device=dev)
    for rows in (hidden[:3, -1], hidden[:, 4095:4096], hidden.view(-1, 4096)[: 5 * 4099 : 4096]):
        rows.copy_(bf16_randn(g, rows.shape).to(dev))
        near = rows.clone(memory_format=torch.contiguous_format)
        assert rows.stride(0) >= 1 << 24
        assert torch.equal(fourbit.matmul(rows, w), fourbit.matmul(near, w)) and torch.equal(fourbit.swiglu(rows, w, w), fourbit.swiglu(near, w, w))
        assert torch.equal(linear(rows), linear(near))
