"""Adapters beside the block linears: selections, and what an adapted linear
takes, keeps and is saved as."""
import pytest
import torch
from torch import nn

from qwen_image_accel import pipeline
from qwen_image_accel.optimizations import adapters as install
from tests import fake_qwen21 as fq
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
