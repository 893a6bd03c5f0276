"""The many-request operators together: captured and replayed, on another stream,
and in the cached-decode block beside the bf16 and MXFP8 profiles."""
import copy

import pytest
import torch

from qwen_image_accel import _native, pipeline
from qwen_image_accel.kernels import adapters as A
from qwen_image_accel.kernels import attention, kv_cache
from qwen_image_accel.optimizations import adapters as install
from qwen_image_accel.optimizations.prefix_cache import QuantizedLayerCache, quantize_layer_cache
from tests import fake_qwen21 as fq
from tests.helpers import bf16_randn, rel_fro


def say(*a):
    print("[case]", *a, flush=True)


def decode_step(dev, b=4, s=3, h=8, hk=2, c=600, r=16, seed=0):
    """A step of drafted tokens: adapted projection -> K/V written -> attention over the cache."""
    g = torch.Generator().manual_seed(seed)
    k = h * 128
    state = dict(x=bf16_randn(g, (b, s, k)).to(dev), base=bf16_randn(g, (b, s, k)).to(dev),
                 down=bf16_randn(g, (3, r, k), k ** -0.5).to(dev), up=bf16_randn(g, (3, k, r)).to(dev),
                 index=torch.tensor([0, -1, 2, 1], dtype=torch.int32, device=dev),
                 lengths=torch.tensor([600, 3, 64, 301], dtype=torch.int32, device=dev),
                 tree=torch.ones(s, s, dtype=torch.bool, device=dev).tril(),
                 new_k=bf16_randn(g, (b, s, hk, 128)).to(dev), new_v=bf16_randn(g, (b, s, hk, 128)).to(dev))
    cache = kv_cache.empty_cache(b, c, hk, 128, dev)
    kv_cache.write_cache(cache, bf16_randn(g, (b, c, hk, 128)).to(dev), bf16_randn(g, (b, c, hk, 128)).to(dev))

    def step():
        q = A.low_rank(state["x"], state["down"], state["up"], state["index"], base=state["base"])
        kv_cache.write_cache(cache, state["new_k"], state["new_v"], start=state["lengths"] - s)
        return attention.attention_cached(q.view(b, s, h, 128), cache, state["lengths"], tree=state["tree"])
    return state, step


@pytest.mark.gpu
def test_captured_step_follows_its_inputs(dev):
    """Two graphs of the step replayed in turn, with eager steps between: new tokens, lengths and adapters are
    read at every replay, and every replay equals the eager result bit for bit."""
    say("graph")
    state, step = decode_step(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    g = torch.Generator().manual_seed(9)
    for i in range(4):
        state["x"].copy_(bf16_randn(g, tuple(state["x"].shape)))
        state["new_k"].copy_(bf16_randn(g, tuple(state["new_k"].shape)))
        state["index"].copy_(torch.tensor([[1, 2, -1, 0], [2, 2, 2, 2], [-1, -1, -1, -1], [0, 1, 2, 7]][i], dtype=torch.int32))
        state["lengths"].copy_(torch.tensor([[599, 5, 64, 300], [40, 41, 600, 3], [3, 3, 3, 3], [600, 600, 600, 600]][i],
                                            dtype=torch.int32))
        want = step()
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        again = step()
        torch.cuda.synchronize()
        for out in (*outs, again):
            assert torch.equal(out, want), i
    del graphs


@pytest.mark.gpu
def test_on_a_stream_of_its_own(dev):
    say("stream")
    _, step = decode_step(dev)
    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [step() for _ in range(3)]
    side.synchronize()
    for out in outs:
        assert torch.equal(out, want)


# ------------------------------------------------------------- in the block --

def _cached(t, inputs, cache=None):
    h, mod, freqs, layer = inputs
    for b in t.transformer_blocks:
        h = b(hidden_states=h, modulation=mod, rotary_emb=freqs, layer_cache=cache or layer, kv_cache_mode="cached")
    return h


def _adapters(t, dim, ffn, names=("a", "b"), paths=None, device="cpu", rank=(8, 24)):
    """Random adapters beside every block linear (or `paths`), strong enough to move the output by some
    ten percent."""
    g = torch.Generator().manual_seed(4)
    out = {}
    for name, r in zip(names, rank):
        out[name] = {}
        for i, block in enumerate(t.transformer_blocks):
            for rel in paths or install.LAYER_GROUPS["all"]:
                m = block.get_submodule(rel)
                out[name][f"transformer_blocks.{i}.{rel}"] = (bf16_randn(g, (r, m.in_features), m.in_features ** -0.5).to(device),
                                                             bf16_randn(g, (m.out_features, r), 0.05).to(device), 0.75)
    return out


def _merged(t, adapter):
    """A copy of t with one adapter added to its bf16 weights."""
    t = copy.deepcopy(t)
    for path, (down, up, scale) in adapter.items():
        _, i, rel = path.split(".", 2)
        m = t.transformer_blocks[int(i)].get_submodule(rel)
        with torch.no_grad():
            m.weight.add_((scale * up.float() @ down.float()).to(m.weight))
    return t


def test_adapters_on_the_cpu_equal_merged_weights():
    """Routing, without kernels: each sequence of the batch runs with its own adapter, as if its weights held it."""
    t = fq.make_transformer(dim=256, heads=2, ffn=512, dtype=torch.float32)
    t.dtype = torch.bfloat16
    ad = _adapters(t, 256, 512)
    merged = {n: _merged(t, ad[n]) for n in ad}
    plain = copy.deepcopy(t)
    inputs = fq.make_inputs(batch=3, dtype=torch.float32)
    route = install.install_adapters(t, ad)
    with torch.no_grad():
        base = _cached(plain, inputs)
        assert torch.equal(_cached(t, inputs), base)                    # nothing selected
        route.select(["b", None, "a"])
        got = _cached(t, inputs)
        for i, ref in enumerate((merged["b"], plain, merged["a"])):
            want = _cached(ref, inputs)[i]
            # fp32 throughout: 1e-3 of the output covers the order of sums
            assert float((got[i] - want).norm() / want.norm()) < 1e-3
        # The gates are tanh of 0.1 N(0, 1), so what the blocks (and the adapters in them) add is small beside the
        # hidden states: the adapters' effect is measured against what the blocks add, and the match against
        # the effect.
        effect = (got[0] - base[0]).norm()
        assert float(effect / (base[0] - inputs[0][0]).norm()) > 1e-2
        assert float((got[0] - _cached(merged["b"], inputs)[0]).norm() / effect) < 1e-2
        route.select(None)
        assert torch.equal(_cached(t, inputs), base)
        install.remove_adapters(t)
        assert torch.equal(_cached(t, inputs), base)
    assert type(t.transformer_blocks[0].attn.to_q) is torch.nn.Linear


def test_each_batch_size_keeps_its_route_tensor():
    """A step captured at one batch size reads the tensor that later selections of that size write."""
    route = install.AdapterRoute(("a", "b"), "cpu")
    route.select(["b", None])
    two = route.index
    route.select(["a"] * 3)
    assert route.index.tolist() == [0, 0, 0]
    route.select(None)
    assert route.index is None
    route.select(["a", "b"])
    assert route.index is two and two.tolist() == [0, 1]


def test_an_adapter_of_rank_zero_adds_nothing():
    stack = install.AdapterStack.of([(torch.zeros(0, 16), torch.zeros(24, 0), 1.0), None], 24, 16, "cpu")
    y = torch.randn(2, 3, 24)
    assert torch.equal(stack.add(torch.randn(2, 3, 16), y.clone(), torch.tensor([0, 1])), y)


def test_adapter_refusals():
    t = fq.make_transformer()
    ok = (torch.zeros(4, 256), torch.zeros(256, 4), 1.0)
    with pytest.raises(ValueError, match="no adapters"):
        install.install_adapters(t, {})
    with pytest.raises(ValueError, match="unknown linears"):
        install.install_adapters(t, {"a": {"transformer_blocks.0.attn.to_x": ok}})
    with pytest.raises(ValueError, match="beside a"):
        install.install_adapters(t, {"a": {"transformer_blocks.0.attn.to_q": (torch.zeros(4, 128), torch.zeros(256, 4), 1.0)}})
    with pytest.raises(ValueError, match="above 128"):
        install.install_adapters(t, {"a": {"transformer_blocks.0.attn.to_q": (torch.zeros(130, 256), torch.zeros(256, 130), 1.0)}})
    assert type(t.transformer_blocks[0].attn.to_q) is torch.nn.Linear  # nothing was replaced
    route = install.install_adapters(t, {"a": {"transformer_blocks.0.attn.to_q": ok}})
    with pytest.raises(RuntimeError, match="once"):
        install.install_adapters(t, {"a": {"transformer_blocks.0.attn.to_q": ok}})
    with pytest.raises(ValueError, match="unknown adapter"):
        route.select(["c"])
    route.select(["a", "a"])
    with pytest.raises(ValueError, match="names 2 sequences"), torch.no_grad():
        _cached(t, fq.make_inputs(batch=1))


@pytest.mark.gpu
@pytest.mark.parametrize("profile", ["fused", "mxfp8"])
def test_block_with_adapters_and_quantized_prefix(dev, profile, monkeypatch):
    """Both profiles, three requests of one batch with their own adapters, over a quantized prefix: each request
    against the same profile alone with the adapter merged into its weights, over the values of that prefix.

    fused: the merged weights are rounded to bf16 once more than the adapter's product, 2^-8 of each weight at most,
    and the activations round at every stage of two blocks: under 2e-2 (a dozen roundings of 2^-8, as a norm a good
    deal less).  mxfp8: the merged weight is quantized to 4 significand bits with the adapter inside it, the unmerged one without:
    two independent roundings of 2^-4 at most per weight, the bar of this profile against bf16 (5e-2) for each side."""
    say("block", profile)
    monkeypatch.setenv("QW21_MXFP8_SKIP_BLOCKS", "")
    t = fq.make_transformer(dim=512, heads=4, ffn=1024, device=dev)
    ad = _adapters(t, 512, 1024, device=dev)
    inputs = fq.make_inputs(dim=512, heads=4, tokens=96, prefix=37, batch=3, device=dev)
    refs = [_merged(t, ad["b"]), copy.deepcopy(t), _merged(t, ad["a"])]
    before = dict(_native.calls)
    quantized = quantize_layer_cache(inputs[3])
    values = fq.LayerCache(*quantized.get())
    with torch.no_grad():
        pipeline.install_hot_path(t, profile, validate=False)
        bare = _cached(t, inputs, quantized)
        route = install.install_adapters(t, ad)
        # One prefix read two ways; the quantized pack rounds q and k once where the bf16 one rounds three times:
        # two roundings of 2^-8 of q and k, a good deal less of the output.
        both = rel_fro(_cached(t, inputs, quantized).float().cpu().numpy(), _cached(t, inputs, values).float().cpu().numpy())
        assert both < 2.0 ** -7
        route.select(["b", None, "a"])
        got = _cached(t, inputs, quantized)
        for i, ref in enumerate(refs):
            pipeline.install_hot_path(ref, profile, validate=False)
            want = _cached(ref, inputs, values)
            delta, change = (got[i] - bare[i]).float(), (want[i] - bare[i]).float()
            err = rel_fro(got[i].float().cpu().numpy(), want[i].float().cpu().numpy())
            assert err < (2e-2 if profile == "fused" else 1e-1), (i, err)
            if i == 1:
                assert torch.equal(got[i], bare[i]) or profile == "mxfp8"
            else:
                assert float(change.norm()) > 0 and float((delta * change).sum() / (delta.norm() * change.norm())) > 0.9
    torch.cuda.synchronize()
    used = {k for k, v in _native.calls.items() if v > before.get(k, 0)}
    assert {"qim_cache_write", "qim_cache_read", "qim_qk_norm_rope_pack_cached", "qim_low_rank"} <= used, used


@pytest.mark.gpu
def test_stacked_qkv_adapters_equal_the_three_alone(dev, monkeypatch):
    """The mxfp8 profile's one call for the stacked Q/K/V against the three linears one by one."""
    from qwen_image_accel.optimizations import decode
    say("stacked qkv")
    monkeypatch.setenv("QW21_MXFP8_SKIP_BLOCKS", "")
    t = fq.make_transformer(dim=512, heads=4, ffn=1024, device=dev)
    with torch.no_grad():
        pipeline.install_hot_path(t, "mxfp8", validate=False)
        route = install.install_adapters(t, _adapters(t, 512, 1024, device=dev))
        route.select(["a", "b"])
        attn = t.transformer_blocks[0].attn
        x = bf16_randn(torch.Generator().manual_seed(1), (2, 40, 512)).to(dev)
        assert attn._adapter_qkv is not None
        got = decode.project_qkv(attn, x, True)
        alone = [getattr(attn, n)(x).unflatten(-1, (4, -1)) for n in ("to_q", "to_k", "to_v")]
    for g, w in zip(got, alone):   # the same GEMM and the same sums, the K split of another width aside: one bf16 step
        assert float((g.float() - w.float()).abs().max() / w.float().abs().max()) < 2.0 ** -7


@pytest.mark.gpu
def test_save_mxfp8_with_adapters_installed(dev, tmp_path, monkeypatch):
    """Saved weights name the linears as without adapters, and load into a fresh transformer."""
    from qwen_image_accel import weights
    say("save with adapters")
    monkeypatch.setenv("QW21_MXFP8_SKIP_BLOCKS", "")
    t = fq.make_transformer(dim=256, heads=2, ffn=512, device=dev)
    fresh = copy.deepcopy(t)
    pipeline.install_hot_path(t, "mxfp8", validate=False)
    paths = weights.save_mxfp8(t, str(tmp_path / "plain.safetensors"))
    install.install_adapters(t, _adapters(t, 256, 512, device=dev))
    assert weights.save_mxfp8(t, str(tmp_path / "w.safetensors")) == paths
    assert weights.load_mxfp8(fresh, str(tmp_path / "w.safetensors")) == paths


@pytest.mark.gpu
def test_quantized_layer_cache(dev):
    say("layer cache")
    g = torch.Generator().manual_seed(0)
    layer = fq.LayerCache(bf16_randn(g, (2, 9, 4, 128)).to(dev), bf16_randn(g, (2, 9, 4, 128)).to(dev))
    q = quantize_layer_cache(layer)
    assert isinstance(q, QuantizedLayerCache) and quantize_layer_cache(q) is q
    for got, x in zip(q.get(), layer.get()):
        assert got.shape == x.shape and float((got.float() - x.float()).abs().max() / x.float().abs().max()) <= 2.0 ** -4
    with pytest.raises(ValueError):
        QuantizedLayerCache(layer.k, layer.v[:, :3])
