"""Adapters beside the block linears: selections, and what an adapted linear
takes, keeps and is saved as."""
import copy
import types

import pytest
import torch
from torch import nn

from qwen_image_accel import _native, pipeline, weights
from qwen_image_accel.optimizations import adapters as install
from qwen_image_accel.optimizations import decode, mxfp8
from qwen_image_accel.optimizations.mxfp8 import MXFP8Linear, quantize_transformer
from tests import fake_qwen21 as fq
from tests import requests_ref as R
from tests.helpers import bf16_randn


def say(*a):
    print("[case]", *a, flush=True)


def adapted(names=("a", "b"), k=64, n=48, r=8, dtype=torch.float32, device="cpu", seed=0):
    """(the linear with its adapters, the linear alone, the route, the stack)."""
    g = torch.Generator().manual_seed(seed)
    base = nn.Linear(k, n, bias=False).to(dtype)
    with torch.no_grad():
        base.weight.copy_(torch.randn(n, k, generator=g) * k ** -0.5)
    base = base.to(device)
    triples = [(torch.randn(r, k, generator=g) * k ** -0.5, torch.randn(n, r, generator=g), 0.5) for _ in names]
    stack = install.AdapterStack.of(triples, n, k, device)
    route = install.AdapterRoute(names, device)
    return install.AdaptedLinear(base, stack, route), base, route, stack


# ------------------------------------------------------------- selections --

def test_a_step_keeps_the_selection_it_was_started_with(monkeypatch):
    """What a later selection writes is nothing that an earlier step may still read."""
    m, _, route, _ = adapted()
    read, add = [], install.AdapterStack.add
    monkeypatch.setattr(install.AdapterStack, "add", lambda self, x, y, index: (read.append(index), add(self, x, y, index))[1])
    x = torch.randn(2, 3, 64)
    with torch.no_grad():
        for names in (["a", None], [None, "b"], ["b", "b"]):
            route.select(names)
            m(x)
    assert [i.tolist() for i in read] == [[0, -1], [-1, 1], [1, 1]]


@pytest.mark.gpu
def test_selections_beside_a_step_on_another_stream(dev):
    """A step queued behind other work on its own stream keeps its selection whatever is selected meanwhile, and a step
    started on another stream after a selection has that one."""
    say("selections and streams")
    m, _, route, _ = adapted(k=256, n=256, dtype=torch.bfloat16, device=dev)
    x = bf16_randn(torch.Generator().manual_seed(1), (2, 40, 256)).to(dev)
    choices = (["a", None], [None, "b"], ["b", "a"], ["b", "b"])
    want, got = [], []
    busy = torch.randn(4096, 4096, device=dev)
    streams = [torch.cuda.Stream() for _ in choices]
    with torch.no_grad():
        for names in choices:
            route.select(names)
            want.append(m(x))
        torch.cuda.synchronize()
        for names, stream in zip(choices, streams):
            route.select(names)
            with torch.cuda.stream(stream):
                for _ in range(8):
                    busy @ busy
                got.append(m(x))
            # Memory of this size that is free on this stream is handed out and written.
            [torch.full((2,), 7, dtype=torch.int32, device=dev) for _ in range(64)]
        torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_switching_off_reaches_captured_steps():
    """A captured step reads the kept tensor of its batch size: nothing selected means no adapter there either."""
    route = install.AdapterRoute(("a", "b"), "cpu")
    route.select(["b", "a", None])
    three = route.index
    route.select(["a", "b"])
    two = route.index
    route.select(None)
    assert route.index is None
    assert three.tolist() == [-1, -1, -1] and two.tolist() == [-1, -1]
    route.select(["b", "b"])
    assert route.index is two and two.tolist() == [1, 1] and three.tolist() == [-1, -1, -1]


@pytest.mark.gpu
def test_captured_layer_follows_selections(dev):
    """Replays of one captured layer across selections, none among them, beside eager calls of the same."""
    say("captured selections")
    m, _, route, _ = adapted(k=256, n=256, dtype=torch.bfloat16, device=dev)
    x = bf16_randn(torch.Generator().manual_seed(1), (2, 40, 256)).to(dev)
    with torch.no_grad():
        route.select(["a", "b"])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m(x)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(x)
        for names in (["b", None], None, ["a", "a"], None, [None, "b"]):
            route.select(names)
            want = m(x)
            torch.cuda.synchronize()
            for _ in range(2):
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, want), names
    del graph


# ------------------------------------------------- what an adapted linear takes --

def shapes():
    """(selection, x's shape, how x is made from a tensor of that shape) for K 64."""
    two, one = ["a", None], ["b"]
    yield "3d", two, lambda r: r(2, 5, 64)
    yield "slice of a batch", two, lambda r: r(2, 9, 64)[:, 4:]
    yield "transposed", two, lambda r: r(5, 2, 64).transpose(0, 1)
    yield "columns", two, lambda r: r(2, 5, 67)[..., 3:]
    yield "columns of aligned rows", two, lambda r: r(2, 5, 80)[..., 4:68]
    yield "4d", two, lambda r: r(2, 3, 4, 64)
    yield "4d slice", two, lambda r: r(2, 3, 4, 64)[:, 1:, ::2]
    yield "expanded", two, lambda r: r(1, 1, 64).expand(2, 5, 64)
    yield "a row per sequence", two, lambda r: r(2, 64)
    yield "rows of one sequence", one, lambda r: r(7, 64)
    yield "one row", one, lambda r: r(64)
    yield "nothing", two, lambda r: r(2, 0, 64)


def check_adapted(m, base, stack, x, names):
    """Against the adapters' definition in float64, one sequence at a time.

    The bound: fp32 sums of K and of R products, off by at most F32 of the sum of magnitudes per addition (16 more for
    the join of chunks, scale and base); h enters the second product as two bf16 terms, HALF^2 of it; the result
    is rounded once, to bf16 or fp32.  The linear's own output is in both sides."""
    with torch.no_grad():
        m.route.select(names)
        got, want = m(x), base(x)
        assert got.shape == want.shape and got.dtype == want.dtype
        rows, index = want.double().reshape(len(names), -1, want.shape[-1]).clone(), m.route.index.tolist()
        xs, bound = x.double().reshape(len(names), -1, x.shape[-1]), torch.zeros_like(rows)
        for i, a in enumerate(index):
            if a >= 0:
                down, up, scale = stack.down[a].double().T, stack.up[a].double().T, float(stack.scale[a])
                rows[i] += scale * (xs[i] @ down) @ up
                bound[i] = ((x.shape[-1] + up.shape[0] + 16) * R.F32 + R.HALF ** 2) * scale * (xs[i].abs() @ down.abs()) @ up.abs()
        half = R.F32 if got.dtype == torch.float32 else R.HALF
        bound += half * (rows.abs() + bound)
        assert ((got.double().reshape(rows.shape) - rows).abs() <= bound).all()


@pytest.mark.parametrize("case", shapes(), ids=lambda c: c[0])
def test_an_adapted_linear_takes_what_the_linear_takes(case):
    _, names, make = case
    m, base, _, stack = adapted()
    g = torch.Generator().manual_seed(3)
    check_adapted(m, base, stack, make(lambda *s: torch.randn(*s, generator=g)), names)


@pytest.mark.gpu
@pytest.mark.parametrize("case", shapes(), ids=lambda c: c[0])
def test_an_adapted_linear_takes_what_the_linear_takes_gpu(dev, case):
    what, names, make = case
    say("adapted linear:", what)
    m, base, _, stack = adapted(dtype=torch.bfloat16, device=dev)
    g = torch.Generator().manual_seed(3)
    check_adapted(m, base, stack, make(lambda *s: torch.randn(*s, generator=g).bfloat16().to(dev)), names)


@pytest.mark.gpu
def test_an_adapted_linear_of_sizes_the_kernel_does_not_take(dev):
    say("adapted linear: K 36, N 52")
    m, base, _, stack = adapted(k=36, n=52, dtype=torch.bfloat16, device=dev)
    x = bf16_randn(torch.Generator().manual_seed(3), (2, 5, 36)).to(dev)
    check_adapted(m, base, stack, x, ["a", None])


def test_rows_that_belong_to_no_sequence_are_refused():
    m, _, route, _ = adapted()
    route.select(["a", None])
    for shape in ((3, 5, 64), (10, 64), (64,)):
        with pytest.raises(ValueError, match="names 2 sequences"), torch.no_grad():
            m(torch.randn(shape))


# ----------------------------------------------- adapters beside some linears --

class HostMXFP8(MXFP8Linear):
    """An MXFP8Linear whose product is the bf16 linear's, for hosts without the kernels."""

    def __init__(self, linear):
        nn.Module.__init__(self)
        self.linear, self.in_features, self.out_features, self.bias = linear, linear.in_features, linear.out_features, None

    def matmul(self, activation):
        return self.linear(activation.rows)

    def forward(self, x):
        return self.linear(x)


def test_an_adapter_beside_the_down_projection_alone(monkeypatch):
    """Gate and value multiply one shared activation into (B * S, F) rows; the adapted down projection still sees
    sequences."""
    mlp = fq.SwiGLU(64, 128)
    plain = copy.deepcopy(mlp)
    for name in ("gate_layer", "proj", "out"):
        setattr(mlp, name, HostMXFP8(getattr(mlp, name)))
    g = torch.Generator().manual_seed(2)
    down, up = torch.randn(8, 128, generator=g) * 0.1, torch.randn(64, 8, generator=g)
    route = install.AdapterRoute(("a",), "cpu")
    mlp.out = install.AdaptedLinear(mlp.out, install.AdapterStack.of([(down, up, 0.5)], 64, 128, "cpu"), route)
    monkeypatch.setattr(decode, "shared_activation", lambda x, consumers: types.SimpleNamespace(rows=x.reshape(-1, 64), shape=x.shape))
    monkeypatch.setattr(decode, "swiglu", lambda gate, value: torch.nn.functional.silu(gate) * value)
    forward, x = decode.QuantizedSwiGLU(mlp), torch.randn(2, 5, 64, generator=g)
    with torch.no_grad():
        want = plain(x)
        assert torch.allclose(forward(x), want, atol=1e-5)      # sums of 128 fp32 products of another order
        route.select(["a", None])
        got = forward(x)
        bf = lambda t: t.bfloat16().float()
        h = torch.nn.functional.silu(plain.gate_layer(x)) * plain.proj(x)
        want[0] += 0.5 * (h[0] @ bf(down).T) @ bf(up).T
        assert torch.allclose(got, want, atol=1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("path", install.LAYER_GROUPS["all"])
def test_mxfp8_block_with_adapters_beside_one_linear(dev, path, monkeypatch):
    """Two requests, one with an adapter on one linear of each block, against the same profile with it merged into the
    weights.  The merged weight is quantized with the adapter inside, 2^-4 of each weight at most and a random part of
    that on average; the adapter is half of the weight's size, so the change it makes points the same way."""
    say("one adapted linear", path)
    monkeypatch.setenv("QW21_MXFP8_SKIP_BLOCKS", "")
    t = fq.make_transformer(dim=512, heads=4, ffn=1024, device=dev)
    ref, ad, g = copy.deepcopy(t), {}, torch.Generator().manual_seed(4)
    for i, block in enumerate(t.transformer_blocks):
        m = block.get_submodule(path)
        down, up = bf16_randn(g, (16, m.in_features), m.in_features ** -0.5), bf16_randn(g, (m.out_features, 16), 0.05)
        ad[f"transformer_blocks.{i}.{path}"] = (down, up, 1.0)
        with torch.no_grad():
            ref.transformer_blocks[i].get_submodule(path).weight.add_((up.float() @ down.float()).to(dev).bfloat16())
    h, mod, freqs, layer = fq.make_inputs(dim=512, heads=4, tokens=96, prefix=37, batch=2, device=dev)
    mod.view(-1, 2, 2, 512)[:, :, 1] *= 10      # gates of O(1): what a block adds is well above the rounding of h

    def run(t):
        x = h
        for b in t.transformer_blocks:
            x = b(hidden_states=x, modulation=mod, rotary_emb=freqs, layer_cache=layer, kv_cache_mode="cached")
        return x.float()
    with torch.no_grad():
        pipeline.install_hot_path(t, "mxfp8", validate=False)
        bare = run(t)
        route = install.install_adapters(t, {"a": ad})
        route.select([None, None])
        none = run(t)
        route.select([None, "a"])
        got = run(t)
        pipeline.install_hot_path(ref, "mxfp8", validate=False)
        want = run(ref)
    assert torch.equal(got[0], none[0])         # the request without an adapter
    delta, change = got[1] - bare[1], want[1] - bare[1]
    assert float((delta * change).sum() / (delta.norm() * change.norm())) > 0.9


# ------------------------------------------------ moved, cast, saved and loaded --

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_adapters_keep_their_types_when_the_model_is_cast(dtype):
    m, _, route, stack = adapted()
    down, up, scale = stack.down.clone(), stack.up.clone(), stack.scale.clone()
    m.to(dtype)
    assert next(m.base.parameters()).dtype == dtype
    for got, want in ((stack.down, down), (stack.up, up), (stack.scale, scale)):
        assert got.dtype == want.dtype and torch.equal(got, want)
    route.select(["a", None])
    with torch.no_grad():
        assert m(torch.randn(2, 3, 64).to(dtype)).dtype == dtype


@pytest.mark.gpu
def test_adapters_move_and_cast_with_the_model(dev):
    """Installed on the host, selected, moved to the GPU, cast, run, captured."""
    say("moved adapters")
    m, base, route, stack = adapted(k=128, n=128)
    route.select(["b", "a"])
    m.to(dev).to(torch.bfloat16)
    x = bf16_randn(torch.Generator().manual_seed(3), (2, 5, 128)).to(dev)
    check_adapted(m, base, stack, x, ["a", None])
    with torch.no_grad():
        want = m(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(x)
        for names in (["a", None], ["b", "b"]):
            route.select(names)
            want = m(x)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
    del graph


@pytest.mark.gpu
def test_a_capture_on_a_device_no_step_ran_on_is_refused(dev):
    say("capture before any step")
    m, _, route, _ = adapted(k=128, n=128)
    route.select(["b", "a"])
    m.to(dev).to(torch.bfloat16)
    x = bf16_randn(torch.Generator().manual_seed(3), (2, 5, 128)).to(dev)
    with torch.no_grad():
        m.base(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            m.base(x)
            with pytest.raises(RuntimeError, match="before it is captured"):
                m(x)
    del graph


def block_with_adapters(mxfp8=()):
    """A block, bf16 but for zero MXFP8 linears at the paths `mxfp8`, and the same with adapters on two of its linears."""
    t = fq.make_transformer(n_blocks=1)
    for path in mxfp8:
        parent, _, leaf = path.rpartition(".")
        m = t.transformer_blocks[0].get_submodule(path)
        codes = torch.arange(m.weight.numel(), dtype=torch.int64).remainder(120).to(torch.uint8).view(m.weight.shape)
        scales = torch.full((m.weight.numel() // 32,), 120, dtype=torch.uint8)
        setattr(t.transformer_blocks[0].get_submodule(parent), leaf,
                MXFP8Linear.from_quantized(m.in_features, m.out_features, codes, scales))
    both = copy.deepcopy(t)
    route = install.install_adapters(both, {"a": {f"transformer_blocks.0.{p}": (torch.randn(4, 256), torch.randn(256, 4), 1.0)
                                                  for p in ("attn.to_q", "attn.to_out.0")}})
    return t, both, route


@pytest.mark.parametrize("mxfp8", [(), ("attn.to_q", "attn.to_k")])
def test_state_dicts_are_those_of_the_model_without_adapters(mxfp8):
    plain, both, _ = block_with_adapters(mxfp8)
    a, b = plain.transformer_blocks.state_dict(), both.transformer_blocks.state_dict()
    assert list(a) == list(b) and a._metadata.keys() >= {"0.attn.to_q", "0.attn.to_out.0"} and a._metadata["0.attn.to_q"] == b._metadata["0.attn.to_q"]
    same = lambda s, t: all(torch.equal(s[k].reshape(-1).view(torch.uint8), t[k].reshape(-1).view(torch.uint8)) for k in s)
    assert same(a, b)
    linear = both.transformer_blocks[0].attn.to_q
    assert list(linear.state_dict()) == list(plain.transformer_blocks[0].attn.to_q.state_dict())
    # Other values, loaded into each from the other.
    other = {k: (v.reshape(-1).view(torch.uint8) ^ 1).view(v.dtype).view(v.shape) for k, v in a.items()}
    both.transformer_blocks.load_state_dict(other)
    assert same(both.transformer_blocks.state_dict(), other)
    plain.transformer_blocks.load_state_dict(both.transformer_blocks.state_dict())
    assert same(plain.transformer_blocks.state_dict(), other)
    key = "0.attn.to_q.weight_fp8" if mxfp8 else "0.attn.to_q.weight"
    linear.load_state_dict({k.removeprefix("0.attn.to_q."): v for k, v in a.items() if k.startswith("0.attn.to_q.")})
    assert same(both.transformer_blocks.state_dict(), {**other, **{k: a[k] for k in a if k.startswith("0.attn.to_q.")}})
    with pytest.raises(RuntimeError, match="Missing key"):
        both.transformer_blocks.load_state_dict({k: v for k, v in a.items() if k != key})
    with pytest.raises(RuntimeError, match="Unexpected key"):
        both.transformer_blocks.load_state_dict({**a, "0.attn.to_q.other": a[key]})


def test_mxfp8_weights_load_beside_adapters(tmp_path):
    """A file saved with or without adapters loads into a transformer with adapters installed, over bf16 and over MXFP8
    linears, the stacked Q/K/V weight among what it restores; the adapters stay."""
    linears = ("attn.to_q", "attn.to_k", "attn.to_v")
    saved, both, route = block_with_adapters(linears)
    weights.fuse_qkv(saved.transformer_blocks[0].attn)
    path = str(tmp_path / "w.safetensors")
    names = weights.save_mxfp8(saved, path)
    assert names == sorted(f"transformer_blocks.0.{p}" for p in linears)
    _, bf16, _ = block_with_adapters()
    for t in (both, bf16):
        attn = t.transformer_blocks[0].attn
        stack = attn.to_q.stack
        assert weights.load_mxfp8(t, path) == names
        assert isinstance(attn.to_q, install.AdaptedLinear) and attn.to_q.stack is stack
        assert isinstance(attn.to_q.base, MXFP8Linear) and isinstance(attn.to_k, MXFP8Linear)
        assert torch.equal(attn.to_q.base.weight_tiled.view(torch.uint8),
                           saved.transformer_blocks[0].attn.to_q.weight_tiled.view(torch.uint8))
        assert torch.equal(attn._mx_qkv[0].view(torch.uint8), saved.transformer_blocks[0].attn._mx_qkv[0].view(torch.uint8))
    again = str(tmp_path / "again.safetensors")
    assert weights.save_mxfp8(both, again) == names and weights.load_mxfp8(saved, again) == names


def test_linears_with_adapters_are_not_silently_left_out_of_the_conversion(monkeypatch):
    """quantize_transformer converts linears; with adapters in front of them it would find none of those."""
    _, both, _ = block_with_adapters()
    with pytest.raises(RuntimeError, match="remove_adapters"):
        quantize_transformer(both, skip_blocks="")
    monkeypatch.setenv("QW21_MXFP8_SKIP_BLOCKS", "")    # its default skips the only block there is
    with pytest.raises(RuntimeError, match="remove_adapters"):
        pipeline.install_hot_path(both, "mxfp8", validate=False)
    assert type(both.transformer_blocks[0].attn.to_k) is nn.Linear and getattr(both, "_qw_hot_path", None) is None
    # Conversions of other linears are as without adapters.
    assert quantize_transformer(both, skip_blocks="0") == []
    monkeypatch.setattr(mxfp8, "MXFP8Linear", HostMXFP8)
    assert quantize_transformer(both, skip_blocks="", layers="mlp") == [f"transformer_blocks.0.img_mlp.{n}" for n in ("gate_layer", "out", "proj")]
    install.remove_adapters(both)
    assert len(quantize_transformer(both, skip_blocks="")) == 4


def test_adapters_of_no_linear_are_refused():
    t = fq.make_transformer(n_blocks=1)
    for adapters in ({"a": {}}, {"a": {}, "b": {}}):
        with pytest.raises(ValueError, match="no adapters"):
            install.install_adapters(t, adapters)
    assert getattr(t, "_qw_adapters", None) is None
    ok = (torch.zeros(4, 256), torch.zeros(256, 4), 1.0)
    route = install.install_adapters(t, {"a": {"transformer_blocks.0.attn.to_q": ok}, "none": {}})   # one of the two is
    route.select(["none"])


# ------------------------------------------------------------- nothing selected --

@pytest.mark.gpu
@pytest.mark.parametrize("profile", ["fused", "mxfp8"])
def test_the_model_runs_without_adapters_while_nothing_is_selected(dev, profile, monkeypatch):
    """The same bits from the same launches as before install_adapters, before a selection and after select(None)."""
    say("nothing selected", profile)
    monkeypatch.setenv("QW21_MXFP8_SKIP_BLOCKS", "")
    monkeypatch.setenv("QW21_ATTENTION_BACKEND", "qim")
    t = fq.make_transformer(dim=512, heads=4, ffn=1024, device=dev)
    h, mod, freqs, layer = fq.make_inputs(dim=512, heads=4, tokens=96, prefix=37, batch=2, device=dev)

    def run():
        before, x = dict(_native.calls), h
        for b in t.transformer_blocks:
            x = b(hidden_states=x, modulation=mod, rotary_emb=freqs, layer_cache=layer, kv_cache_mode="cached")
        return x, {k: n - before.get(k, 0) for k, n in _native.calls.items() if n != before.get(k, 0)}
    with torch.no_grad():
        pipeline.install_hot_path(t, profile, validate=False)
        bare, launches = run()
        bare, launches = run()
        ad = {}
        for i, block in enumerate(t.transformer_blocks):
            for path in install.LAYER_GROUPS["all"]:
                m = block.get_submodule(path)
                ad[f"transformer_blocks.{i}.{path}"] = (torch.randn(8, m.in_features), torch.randn(m.out_features, 8), 0.1)
        route = install.install_adapters(t, {"a": ad})
        for names in (None, ["a", None], None):
            route.select(names)
            out, used = run()
            if names is None:
                assert torch.equal(out, bare) and used == launches
            else:
                assert not torch.equal(out, bare) and used["qim_low_rank"] > 0


@pytest.mark.gpu
@pytest.mark.parametrize("profile", ["fused", "mxfp8"])
def test_a_request_without_adapters_does_not_see_its_neighbours(dev, profile, monkeypatch):
    """Every linear adapted: the request without an adapter gives the same bits whatever the others have, none among them."""
    say("no adapter beside adapters", profile)
    monkeypatch.setenv("QW21_MXFP8_SKIP_BLOCKS", "")
    t = fq.make_transformer(dim=512, heads=4, ffn=1024, device=dev)
    h, mod, freqs, layer = fq.make_inputs(dim=512, heads=4, tokens=96, prefix=37, batch=3, device=dev)
    g, ad = torch.Generator().manual_seed(8), {"a": {}, "b": {}}
    for i, block in enumerate(t.transformer_blocks):
        for path in install.LAYER_GROUPS["all"]:
            m = block.get_submodule(path)
            for name, r in (("a", 8), ("b", 24)):
                ad[name][f"transformer_blocks.{i}.{path}"] = (bf16_randn(g, (r, m.in_features)), bf16_randn(g, (m.out_features, r)), 0.1)
    with torch.no_grad():
        pipeline.install_hot_path(t, profile, validate=False)
        route = install.install_adapters(t, ad)
        outs = []
        for names in ([None, None, None], ["a", None, "b"], ["b", None, "b"], ["a", None, None]):
            route.select(names)
            x = h
            for b in t.transformer_blocks:
                x = b(hidden_states=x, modulation=mod, rotary_emb=freqs, layer_cache=layer, kv_cache_mode="cached")
            outs.append(x)
    for out in outs[1:]:
        assert torch.equal(out[1], outs[0][1]) and not torch.equal(out[0], outs[0][0])
    assert torch.equal(outs[3][2], outs[0][2]) and torch.equal(outs[1][2], outs[2][2])
