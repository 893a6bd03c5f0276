"""The joined residual and norm of the cached-decode block: no slower than the two calls that it replaces, with their bits."""
import pytest
import torch

from qwen_image_accel.kernels import elementwise, epilogue, layernorm
from tests.helpers import bf16_randn

pytestmark = pytest.mark.gpu


def calls(d, quantized):
    norm = torch.nn.LayerNorm(d, eps=1e-6, elementwise_affine=False)

    def parts(h, x, gate, scale):
        h = elementwise.residual(h, x, gate)
        return h, epilogue.layer_norm_scale_quantize(h, scale, norm, tiled=True) if quantized else layernorm.layer_norm_scale(h, scale, norm)

    def joined(h, x, gate, scale):
        return elementwise.residual_norm(h, x, norm, gate=gate, scale=scale, quantized=quantized, tiled=quantized, rounding="eager")
    return parts, joined


def same(a, b):
    if not isinstance(a, torch.Tensor):
        return torch.equal(a.values.view(torch.uint8), b.values.view(torch.uint8)) and torch.equal(a.scales.view(torch.uint8), b.scales.view(torch.uint8))
    return torch.equal(a, b)


@pytest.mark.parametrize("b,s,d", [(1, 7, 4104), (2, 33, 4352), (1, 64, 4608), (1, 5, 6152), (1, 9, 7680), (3, 50, 8192), (1, 2, 8200)])
def test_bits(dev, b, s, d):
    print("[case] joined bits", b, s, d, flush=True)
    g = torch.Generator().manual_seed(d)
    h, x = bf16_randn(g, (b, s, d), 2.0).to(dev), bf16_randn(g, (b, s, d)).to(dev)
    gate, scale = bf16_randn(g, (b, 1, d)).to(dev), bf16_randn(g, (b, 1, d)).to(dev)
    h[0, 1] = 3.0 + h[0, 1] / 512                       # a mean far from 0: the variance's second pass
    for quantized in (False, True) if d % 128 == 0 else (False,):
        parts, joined = calls(d, quantized)
        want, got = parts(h, x, gate, scale), joined(h, x, gate, scale)
        assert torch.equal(got[0], want[0]) and same(got[1], want[1])


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("d", [1024, 4096, 4608, 6144, 8192, 16384])
def test_no_slower_than_two_calls(dev, d, quantized):
    """Times of 4096 rows, the least of nine replays of twelve calls on inputs that no cache holds."""
    print("[case] joined time", d, quantized, flush=True)
    sets = []
    for i in range(4):
        h, x = (torch.randn(1, 4096, d, device=dev).to(torch.bfloat16) for _ in range(2))
        gate, scale = (torch.randn(1, 1, d, device=dev).to(torch.bfloat16) for _ in range(2))
        sets.append((h, x, gate, scale))
    best, graphs = [], []
    for f in calls(d, quantized):
        f(*sets[0])
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            for i in range(12):
                f(*sets[i % 4])
        best.append(float("inf"))
    for _ in range(9):
        for i, graph in enumerate(graphs):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            graph.replay()
            end.record()
            torch.cuda.synchronize()
            best[i] = min(best[i], start.elapsed_time(end))
    print("two calls %.1f us, joined %.1f us" % tuple(1000 / 12 * t for t in best), flush=True)
    assert best[1] <= 1.05 * best[0]
