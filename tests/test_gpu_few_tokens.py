"""The operators of a step of a few tokens together: a decoder layer whose requests continue shared prefixes, its
projections in 4 bits, its residuals joined with its norms; and the cached-decode block with the joined pass."""
import types

import pytest
import torch

from qwen_image_accel import _native
from qwen_image_accel.kernels import attention, elementwise, fourbit, kv_cache
from qwen_image_accel.optimizations import decode
from qwen_image_accel import pipeline
from tests import fake_qwen21 as fq
from tests import few_tokens_ref as R
from tests.helpers import bf16_randn

pytestmark = pytest.mark.gpu

DIM, HEADS, KV, FFN, HEAD = 512, 4, 2, 768, 128


def say(*a):
    print("[case]", *a, flush=True)


class Layer:
    """h -> norm, Q/K/V, cache, attention, out projection, residual and norm, SwiGLU, down projection, residual and norm."""

    def __init__(self, dev, requests, seq, capacity, share, prefix_lengths, prefix):
        g = torch.Generator().manual_seed(3)

        def weight(n, k, **kw):
            return fourbit.quantize_weight(torch.randn(n, k, generator=g) * k ** -0.5, **kw)

        def norm():
            return types.SimpleNamespace(weight=(1 + 0.1 * bf16_randn(g, (DIM,))).to(torch.bfloat16).to(dev), bias=None, eps=1e-6)
        ws = dict(qkv=weight((HEADS + 2 * KV) * HEAD, DIM, kind="int4", group=64), out=weight(DIM, HEADS * HEAD, kind="mxfp4"),
                  gate=weight(FFN, DIM, kind="int4", group=128, symmetric=True), up=weight(FFN, DIM, kind="int4", group=128, symmetric=True),
                  down=weight(DIM, FFN, kind="int4", group=32))
        self.w = {k: v._replace(codes=v.codes.to(dev), scales=v.scales.to(dev), zeros=None if v.zeros is None else v.zeros.to(dev))
                  for k, v in ws.items()}
        self.norms = [norm() for _ in range(5)]
        self.seq, self.share, self.plens = seq, share, prefix_lengths
        self.prefix = kv_cache.empty_cache(len(prefix_lengths), prefix, KV, HEAD, dev)
        kv_cache.write_cache(self.prefix, *(bf16_randn(g, (len(prefix_lengths), prefix, KV, HEAD)).to(dev) for _ in range(2)))
        self.cache = kv_cache.empty_cache(requests, capacity, KV, HEAD, dev)
        for t in self.cache:
            t.view(torch.uint8).zero_()

    def step(self, h, start, tree, keep=None):
        n0, post1, n1, post2, n2 = self.norms
        zero = torch.zeros_like(h)
        _, x = elementwise.residual_norm(h, zero, n0)
        qkv = fourbit.matmul(x, self.w["qkv"]).unflatten(-1, (-1, HEAD))
        q, k, v = qkv[:, :, :HEADS], qkv[:, :, HEADS:HEADS + KV], qkv[:, :, HEADS + KV:]
        kv_cache.write_cache(self.cache, k, v, start=start)
        lengths = start + self.seq
        o = attention.attention_shared(q, self.prefix, self.cache, lengths, share=self.share, prefix_lengths=self.plens, tree=tree)
        y = fourbit.matmul(o.flatten(2), self.w["out"])
        h1, x1 = elementwise.residual_norm(h, y, n1, post=post1)
        a = fourbit.swiglu(x1, self.w["gate"], self.w["up"])
        d = fourbit.matmul(a, self.w["down"])
        h2, x2 = elementwise.residual_norm(h1, d, n2, post=post2)
        if keep is not None:
            keep.update(x=x, qkv=qkv, lengths=lengths, o=o, y=y, h1=h1, x1=x1, a=a, d=d, h2=h2, x2=x2)
        return h2, x2


def make(dev, seq):
    share = torch.tensor([0, 1, 0, -1, 1, 0], dtype=torch.int32, device=dev)
    plens = torch.tensor([70, 33], dtype=torch.int32, device=dev)
    layer = Layer(dev, 6, seq, 24, share, plens, 70)
    g = torch.Generator().manual_seed(5)
    tree = torch.ones(seq, seq, dtype=torch.bool).tril().to(dev)
    return layer, [bf16_randn(g, (6, seq, DIM)).to(dev) for _ in range(3)], tree, torch.tensor([0, 2, 4, 1, 0, 3], dtype=torch.int32, device=dev)


def rms(n):
    return ("rms", n.weight, n.eps)


def inside(got, want, bound):
    err = (got.reshape(want.shape).double().cpu() - want).abs()
    assert got.isfinite().all() and (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("seq", [1, 5])
def test_a_layer_step_by_step(dev, seq):
    """Every stage against float64 on what the stage before gave."""
    say("layer", seq)
    layer, hs, tree, start = make(dev, seq)
    n0, post1, n1, post2, n2 = layer.norms
    for h in hs:
        keep = {}
        layer.step(h, start, tree, keep)

        def four(x, name):
            return R.four_bit(x.reshape(-1, x.shape[-1]), *fourbit.unpack_weight(layer.w[name]))
        _, _, z, ez = R.residual_norm(h, torch.zeros_like(h), rms(n0))
        inside(keep["x"], z, R.rounded(z, ez))
        y, e = four(keep["x"], "qkv")
        inside(keep["qkv"], y, R.rounded(y, e))
        o, bound = R.attention_shared(keep["qkv"][:, :, :HEADS], kv_cache.read_cache(layer.prefix), kv_cache.read_cache(layer.cache),
                                      keep["lengths"].tolist(), layer.share.tolist(), layer.plens.tolist(), tree)
        inside(keep["o"], o, bound)
        y, e = four(keep["o"].flatten(2), "out")
        inside(keep["y"], y, R.rounded(y, e))
        for h_in, x, post, norm, out, z_out in ((h, keep["y"], post1, n1, "h1", "x1"), (keep["h1"], keep["d"], post2, n2, "h2", "x2")):
            hw, bh, z, ez = R.residual_norm(h_in, x, rms(norm), post=rms(post))
            inside(keep[out], hw, bh)
            inside(keep[z_out], z, R.rounded(z, ez))
        y, e = R.swiglu(four(keep["x1"], "gate"), four(keep["x1"], "up"))
        inside(keep["a"], y, R.rounded(y, e))
        y, e = four(keep["a"], "down")
        inside(keep["d"], y, R.rounded(y, e))
        start += seq


def test_a_captured_layer(dev):
    """The step in a graph, its start advanced between the replays, against eager steps."""
    say("captured layer")
    layer, hs, tree, start = make(dev, 5)
    first = start.clone()
    want = []
    for h in hs:
        want.append([t.clone() for t in layer.step(h, start, tree)])
        start += 5
    for t in layer.cache:
        t.view(torch.uint8).zero_()
    start.copy_(first)
    h = hs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.step(h, start, tree)
    for i in range(3):
        h.copy_(hs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[i][0]) and torch.equal(got[1], want[i][1]), i
        start += 5


@pytest.mark.parametrize("profile", ["fused", "mxfp8"])
@pytest.mark.parametrize("tokens,batch", [(200, 1), (64, 2), (1, 3)])
def test_cached_decode_keeps_its_bits(dev, profile, tokens, batch, monkeypatch):
    """The cached-decode block with the residual and norm2 in one pass, and with the two launches."""
    say("decode", profile, tokens, batch)
    monkeypatch.setenv("QW21_MXFP8_SKIP_BLOCKS", "")
    t = fq.make_transformer(dim=512, heads=4, ffn=1024, device=dev)
    h, mod, freqs, cache = fq.make_inputs(dim=512, heads=4, tokens=tokens, prefix=37, batch=batch, device=dev)
    pipeline.install_hot_path(t, profile, validate=False)

    def run():
        x = h
        with torch.no_grad():
            for block in t.transformer_blocks:
                x = block(hidden_states=x, modulation=mod, rotary_emb=freqs, layer_cache=cache, kv_cache_mode="cached")
        return x
    before = _native.calls.get("qim_residual_norm", 0)
    joined = run()
    assert _native.calls.get("qim_residual_norm", 0) == before + len(t.transformer_blocks)
    monkeypatch.setattr(decode, "MAX_JOINED_ROWS", 0)
    parts = run()
    assert _native.calls.get("qim_residual_norm", 0) == before + len(t.transformer_blocks)
    assert torch.equal(joined, parts)


def test_two_calls_at_once(dev):
    """The same operators on two streams at the same time, with inputs, weights and caches in common."""
    say("two streams")
    g = torch.Generator().manual_seed(5)
    w = [fourbit.quantize_weight(bf16_randn(g, (1500, 1024)).to(dev).float(), "int4", 64) for _ in range(2)]
    x, h = (bf16_randn(g, (2, 40, 1024)).to(dev) for _ in range(2))
    caches = []
    for b, c in ((2, 900), (40, 30)):
        caches.append(kv_cache.empty_cache(b, c, 4, 128, dev))
        kv_cache.write_cache(caches[-1], bf16_randn(g, (b, c, 4, 128)).to(dev), bf16_randn(g, (b, c, 4, 128)).to(dev))
    q, n = bf16_randn(g, (40, 2, 8, 128)).to(dev), torch.full((40,), 30, dtype=torch.int32, device=dev)
    share, norm = torch.arange(40, dtype=torch.int32, device=dev) % 3 - 1, torch.nn.RMSNorm(1024, eps=1e-6, device=dev, dtype=torch.bfloat16)

    def step():
        return (fourbit.swiglu(x, *w), fourbit.matmul(x[0, :3], w[0]), attention.attention_shared(q, *caches, n, share=share),
                *elementwise.residual_norm(h, x, norm))
    want = step()
    streams, results = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        for s, r in zip(streams, results):
            with torch.cuda.stream(s):
                r.append(step())
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for got in r for a, b in zip(got, want))
