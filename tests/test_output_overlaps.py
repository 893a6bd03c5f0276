"""Outputs of the few-token operators over inputs that other workgroups still read: refused before any launch (no GPU), and
outputs between such inputs are taken (GPU)."""
import pytest
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import elementwise, fourbit
from tests.helpers import bf16_randn
from tests.test_few_tokens_refusals import ARG, FAR, four, norm, share

FREE = 64 * FAR    # an address far from all others
HO, Z = 3 * FAR, 4 * FAR


@pytest.mark.parametrize("call", [
    # h' over the vectors: the first, one of a later sequence, a part of one, one that begins in the gap before a row
    norm(gate=HO), norm(gate=HO - 2 * 256), norm(gate=HO + 7 * 512), norm(scale=HO + 16), norm(shift=HO + 512), norm(gate=HO - 496, gate_b=0),
    norm(gate=HO + 1024, ldho=512, gate_b=0), norm(gate=HO + 512 + 16, ldho=512, gate_b=0), norm(gate=HO - 1024, gate_b=512),
    norm(norm=1, norm_w=HO + 512), norm(post=1, post_w=HO + 512),
    # z over them, as rows and as codes and exponents
    norm(gate=Z), norm(scale=Z + 7 * 512), norm(shift=Z - 496), norm(norm=1, norm_w=Z), norm(gate=Z, zs=FREE),
    norm(shift=Z + 128 * 256 - 16, zs=FREE), norm(scale=FREE + 16, zs=FREE)])
def test_residual_norm_refuses(call):
    name, args = call
    rc = getattr(_native.lib(), name)(*args)
    assert rc == ARG, (rc, _native.lib().qim_last_error())


def attend(places, **kw):
    """A call of qim_attention_shared whose operands lie far from each other, except for those placed here."""
    name, args = share(**kw)
    args = list(args)
    for i, at in enumerate((0, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 16, 17)):
        if args[at] is not None:
            args[at] = (8 + 2 * i) * FAR
    for at, value in places.items():
        args[at] = value
    return name, args


Q, O, WS = 8 * FAR, (8 + 2 * 13) * FAR, (8 + 2 * 14) * FAR
OUT = 2 * 2 * 1 * 4 * 128           # bytes of o
CODES = 3 * 64 * 2 * 128            # of a prefix cache


@pytest.mark.parametrize("places,kw", [
    ({0: O}, {}), ({3: O}, {}), ({3: O - CODES + 16}, {}), ({4: O}, {}), ({4: O - CODES // 32 + 16}, {}), ({5: O + OUT - 16}, {}), ({6: O + 16}, {}),
    ({7: O + OUT - 4}, {}), ({8: O - 4}, {}), ({9: O}, {}), ({10: O}, {}), ({11: O - 2 * 32 * 2 * 128 + 16}, {}), ({12: O + 32}, {}), ({13: O + 4}, {}),
    ({14: O}, dict(tree=16)), ({17: O}, {}), ({16: WS + 4096}, {}), ({0: WS}, {}), ({3: WS + 256}, {}), ({13: WS + 8}, {}), ({8: WS + 512}, {})])
def test_attention_shared_refuses(places, kw):
    name, args = attend(places, **kw)
    rc = getattr(_native.lib(), name)(*args)
    assert rc == ARG and b"overlap" in _native.lib().qim_last_error(), (rc, _native.lib().qim_last_error())


# A weight of 100 rows and 256 k: 7 tiles of 2 steps.
W4 = dict(m=4, n=100, k=256, ldo=100, zeros=5 * FAR, codes=6 * FAR, scales=7 * FAR)
GATE_UP = dict(W4, codes2=8 * FAR, scales2=9 * FAR, zeros2=10 * FAR)


@pytest.mark.parametrize("call", [
    four(**W4 | dict(out=6 * FAR)), four(**W4 | dict(out=6 * FAR + 14 * 1024 - 16)), four(**W4 | dict(out=7 * FAR + 14 * 64 - 2)),
    four(**W4 | dict(out=5 * FAR - 798)), four(**W4 | dict(out=5 * FAR + 14 * 32 - 16)), four(**GATE_UP | dict(out=8 * FAR)),
    four(**GATE_UP | dict(out=9 * FAR - 2)), four(**GATE_UP | dict(out=10 * FAR)), four(**W4 | dict(bias=2 * FAR + 200)),
    four(**W4 | dict(bias=2 * FAR + 799 - 1)), four(**W4 | dict(bias=2 * FAR - 198)), four(**W4 | dict(bias=2 * FAR + 4 * 396, ldo=300, f32=1)),
    four(**dict(W4, zeros=None, group=0) | dict(out=7 * FAR + 14 * 64 - 2)), four(**dict(W4, group=32) | dict(out=7 * FAR + 14 * 128 - 2))])
def test_fourbit_refuses(call):
    name, args = call
    rc = getattr(_native.lib(), name)(*args)
    assert rc == ARG and b"overlap" in _native.lib().qim_last_error(), (rc, _native.lib().qim_last_error())


@pytest.mark.gpu
def test_a_bias_beside_the_rows_of_one_buffer(dev):
    print("[case] bias beside rows", flush=True)
    g = torch.Generator().manual_seed(1)
    w = fourbit.quantize_weight(bf16_randn(g, (40, 128)).to(dev))
    x, bias = bf16_randn(g, (6, 128)).to(dev), bf16_randn(g, (40,)).to(dev)
    want = fourbit.matmul(x, w, bias=bias)
    wide = torch.zeros(6, 100, dtype=torch.bfloat16, device=dev)
    wide[3, 50:90] = bias
    got = fourbit.matmul(x, w, bias=wide[3, 50:90], out=wide[:, 3:43])
    assert torch.equal(got, want) and torch.equal(wide[3, 50:90], bias)
    with pytest.raises(_native.QimError):
        fourbit.matmul(x, w, bias=wide[3, 40:80], out=wide[:, 3:43])


@pytest.mark.gpu
def test_vectors_beside_the_rows_of_one_buffer(dev):
    """gate, scale and shift in other columns of the buffer that h' goes to, and behind its last row."""
    print("[case] vectors beside rows", flush=True)
    g = torch.Generator().manual_seed(1)
    b, s, d = 3, 5, 264
    h, x = (bf16_randn(g, (b, s, d)).to(dev) for _ in range(2))
    layer = torch.nn.LayerNorm(d, eps=1e-6, elementwise_affine=False)
    vectors = {k: bf16_randn(g, (b, 1, d)).to(dev) for k in ("gate", "scale", "shift")}
    want = elementwise.residual_norm(h, x, layer, **vectors)
    wide = torch.zeros(b * s + 1, 4 * d, dtype=torch.bfloat16, device=dev)
    out = wide[:b * s].view(b, s, 4 * d)[..., :d]
    places = {k: wide[:b * s].view(b, s, 4 * d)[:, 2:3, (i + 1) * d:(i + 2) * d] for i, k in enumerate(vectors)}
    for k, v in vectors.items():
        places[k].copy_(v)
    got = elementwise.residual_norm(h, x, layer, out=out, **places)
    assert got[0] is out and torch.equal(out, want[0]) and torch.equal(got[1], want[1])
    assert all(torch.equal(places[k], v) for k, v in vectors.items())
    last = wide[b * s, :d]
    last.copy_(vectors["gate"][0, 0])
    one = dict(vectors, gate=last)
    want = elementwise.residual_norm(h, x, layer, **dict(vectors, gate=vectors["gate"][0, 0].clone()))
    got = elementwise.residual_norm(h, x, layer, out=out, **one)
    assert torch.equal(out, want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(_native.QimError):
        elementwise.residual_norm(h, x, layer, out=out, **dict(vectors, gate=wide[1, :d]))
