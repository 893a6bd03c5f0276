"""Low-rank adapters on the block linears, chosen per request.

``install_adapters`` puts any number of named adapters beside the (bf16 or
MXFP8) linears of a transformer, after ``install_hot_path``; each batch then
names the adapter of every sequence with ``AdapterRoute.select``, so that one
model serves requests with different adapters (or none) together, without
merging weights.  The reference has no adapters; there is no reference
counterpart.
"""
import torch
from torch import nn

from qwen_image_accel import _native
from qwen_image_accel.kernels.adapters import MAX_RANK, low_rank, takes_rows
from qwen_image_accel.optimizations.mxfp8 import LAYER_GROUPS, MXFP8Linear
from qwen_image_accel.weights import ADAPTED_BASE

NO_ADAPTER = -1


class AdapterRoute:
    """Which adapter each sequence of the batch uses, an adapter's number or -1;
    nothing while nothing is selected (no adapter anywhere).

    A step reads a tensor that its selection wrote before ``select`` returned
    and that nothing writes again: a step already queued keeps its selection,
    and one started afterwards, on any stream, has the new one.  A step that is
    captured into a graph reads a kept tensor instead (``index``, on the device the adapters were
    installed on): each batch size has one, from its first ``select``
    on, written by the later ones of that batch size
    on the current stream, as any other input of a graph is
    (order replays on another stream behind it, and ``select`` behind them)."""

    def __init__(self, names, device):
        self.names, self.device, self.index = tuple(names), torch.device(device), None
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._kept = {self.device: {}}  # per device that a step ran on: batch size -> tensor
        self._numbers, self._steps = None, {}

    def select(self, names):
        """``names``: one adapter name (or None) per sequence of the batch;
        or None to switch the adapters off, in captured steps of every batch
        size too.  (A step captured while nothing was selected has no adapters in
        it, whatever is selected later.)"""
        if names is None:
            self.index, self._numbers, self._steps = None, None, {}
            for by_batch in self._kept.values():
                for kept in by_batch.values():
                    kept.fill_(NO_ADAPTER)
            return
        numbers = []
        for name in names:
            if name is not None and name not in self.names:
                raise ValueError(f"unknown adapter {name!r}; installed: {list(self.names)}")
            numbers.append(NO_ADAPTER if name is None else self.names.index(name))
        self._numbers, self._steps = numbers, {}
        for device in self._kept:
            self._write(device)
        self.index = self._kept[self.device][len(numbers)]

    def _write(self, device):
        """The selection on `device`: its own tensor, and the kept one of its batch size."""
        step, by_batch = torch.tensor(self._numbers, dtype=torch.int32, device=device), self._kept[device]
        self._steps[device] = step, set()
        if len(self._numbers) in by_batch:
            by_batch[len(self._numbers)].copy_(step)
        else:
            by_batch[len(self._numbers)] = step.clone()

    @property
    def off(self):
        """Whether nothing is selected."""
        return self._numbers is None

    def step_index(self, device):
        """The int32 (B,) tensor on `device` that a step started now reads, or None."""
        if self.off:
            return None
        capturing = device.type == "cuda" and torch.cuda.is_current_stream_capturing()
        if device not in self._steps:  # the model was moved, or has linears on several devices
            if capturing:
                raise RuntimeError(f"run the adapted step once on {device} before it is captured")
            self._kept.setdefault(device, {})
            self._write(device)
        if capturing:
            return self._kept[device][len(self._numbers)]
        step, streams = self._steps[device]
        if device.type == "cuda":
            stream = _native.stream(device)
            if stream not in streams:  # its memory outlives what this stream does with it
                streams.add(stream)
                step.record_stream(torch.cuda.current_stream(device))
        return step


class AdapterStack(nn.Module):
    """The adapters of one projection, stacked: down (A, parts * R, K), up (A, N,
    R) in bf16, scale (A,).  An adapter of a smaller rank is padded with zeros, one that
    does not touch this projection is zeros with scale 0.  The three keep their
    types when the model around them is cast."""

    def __init__(self, down, up, scale, parts=1):
        super().__init__()
        self.parts = parts
        self.register_buffer("down", down, persistent=False)
        self.register_buffer("up", up, persistent=False)
        self.register_buffer("scale", scale, persistent=False)

    def _apply(self, fn, recurse=True):
        kept = dict(self.named_buffers(recurse=False))
        super()._apply(fn, recurse)
        for name, t in kept.items():
            moved = getattr(self, name)
            if moved.dtype != t.dtype:
                setattr(self, name, t.to(moved.device))
        return self

    @classmethod
    def of(cls, triples, out_features, in_features, device):
        """``triples``: per adapter (down (r, K), up (N, r), scale) or None."""
        ranks = [t[0].shape[0] for t in triples if t is not None]
        r = max(8, (max(ranks) + 7) // 8 * 8)
        if r > MAX_RANK:
            raise ValueError(f"adapter rank {max(ranks)} is above {MAX_RANK}")
        down = torch.zeros(len(triples), r, in_features, dtype=torch.bfloat16, device=device)
        up = torch.zeros(len(triples), out_features, r, dtype=torch.bfloat16, device=device)
        scale = torch.zeros(len(triples), dtype=torch.float32, device=device)
        for i, t in enumerate(triples):
            if t is None:
                continue
            d, u, s = t
            if d.dim() != 2 or u.dim() != 2 or d.shape[1] != in_features or u.shape != (out_features, d.shape[0]):
                raise ValueError(f"adapter of shapes {tuple(d.shape)}, {tuple(u.shape)} beside a "
                                 f"({out_features}, {in_features}) linear")
            down[i, :d.shape[0]] = d.to(device=device, dtype=torch.bfloat16)
            up[i, :, :d.shape[0]] = u.to(device=device, dtype=torch.bfloat16)
            scale[i] = float(s)
        return cls(down, up, scale)

    def add(self, x, y, index):
        """y + the adapters' share of x; y may be overwritten.

        x (..., K), y (..., N): the leading axis is the sequences (so a 2-D x holds a
        row of each); of a batch of one, x may be its rows alone or one row."""
        lead, b = x.shape[:-1], index.shape[0]
        if not (lead[:1] == (b,) or (b == 1 and len(lead) < 2)):
            raise ValueError(f"the route names {b} sequences, the batch is {tuple(x.shape)}")
        k, n = x.shape[-1], y.shape[-1]
        if 0 in lead:
            return y
        xs, out = x.reshape(b, -1, k), y.reshape(b, -1, n)
        if (x.is_cuda and x.dtype == torch.bfloat16 and y.dtype == torch.bfloat16
                and k % 8 == 0 and n % (8 * self.parts) == 0):
            # Rows that the kernel does not take as they lie (a slice of a batch) are copied, as the linear does.
            xs, out = (t if takes_rows(t) else t.clone(memory_format=torch.contiguous_format) for t in (xs, out))
            return low_rank(xs, self.down, self.up, index, scale=self.scale, base=out, out=out, parts=self.parts).reshape(y.shape)
        out, r = out.float(), self.up.shape[2]
        for i, a in enumerate(index.tolist()):
            if a >= 0:
                h = (xs[i].float() @ self.down[a].float().t()).unflatten(-1, (self.parts, r))
                up = self.up[a].float().unflatten(0, (self.parts, -1))
                out[i] += self.scale[a] * torch.einsum("spr,pnr->spn", h, up).flatten(1)
        return out.to(y.dtype).reshape(y.shape)


class AdaptedLinear(nn.Module):
    """A linear (nn.Linear or MXFP8Linear) with adapters beside it.  A state dict
    holds the linear under its own path, as without adapters."""

    def __init__(self, base, stack, route):
        super().__init__()
        self.add_module(ADAPTED_BASE, base)
        self.stack, self.route = stack, route
        self.in_features, self.out_features = base.in_features, base.out_features

    @property
    def base(self):
        return getattr(self, ADAPTED_BASE)

    def forward(self, x):
        y, index = self.base(x), self.route.step_index(x.device)
        return y if index is None else self.stack.add(x, y, index)

    def state_dict(self, *args, **kwargs):
        return self.base.state_dict(*args, **kwargs)

    def _load_from_state_dict(self, state_dict, prefix, *args, **kwargs):
        inner = f"{prefix}{ADAPTED_BASE}."
        for key in [k for k in state_dict if k.startswith(prefix) and not k.startswith(inner)]:
            state_dict[inner + key[len(prefix):]] = state_dict.pop(key)
        super()._load_from_state_dict(state_dict, prefix, *args, **kwargs)


def running(linear):
    """The module that a step started now runs at a linear's place: the linear
    itself while nothing is selected, so that the paths which fuse several MXFP8
    linears or their neighbours see them as without adapters."""
    return linear.base if isinstance(linear, AdaptedLinear) and linear.route.off else linear


def _stacked_qkv(linears):
    """One AdapterStack over the stacked Q/K/V projection, or None where the
    three do not stack."""
    if not all(isinstance(m, AdaptedLinear) and isinstance(m.base, MXFP8Linear) for m in linears):
        return None
    stacks = [m.stack for m in linears]
    if len({s.up.shape for s in stacks}) != 1 or not all(torch.equal(s.scale, stacks[0].scale) for s in stacks):
        return None
    return AdapterStack(torch.cat([s.down for s in stacks], 1), torch.cat([s.up for s in stacks], 1), stacks[0].scale,
                        parts=3)


def install_adapters(transformer, adapters):
    """Put named adapters beside the block linears, once, after
    ``install_hot_path``.

    ``adapters``: {name: {path: (down (r, K), up (N, r), scale)}}, ``path`` as
    ``quantize_transformer`` returns them ("transformer_blocks.<i>.attn.to_q";
    any of LAYER_GROUPS["all"]), scale the factor on up @ down (alpha / rank).
    Ranks up to 128 may differ; down and up are held in bf16.  Returns the ``AdapterRoute``; until its
    ``select`` names adapters the model runs without them, as before.  With a selection
    the mxfp8 profile's steps around an adapted linear run one by one: its
    input is normalised in bf16 and quantized for it, gate and up are two
    GEMMs and a SwiGLU, the attention's output is bf16."""
    if getattr(transformer, "_qw_adapters", None) is not None:
        raise RuntimeError("adapters are installed once per transformer; remove_adapters first")
    if not any(adapters.values()):
        raise ValueError("no adapters given")
    names = list(adapters)
    blocks = transformer.transformer_blocks
    known = {f"transformer_blocks.{i}.{p}": (i, p) for i in range(len(blocks)) for p in LAYER_GROUPS["all"]}
    paths = sorted({p for a in adapters.values() for p in a})
    unknown = [p for p in paths if p not in known]
    if unknown:
        raise ValueError(f"adapters for unknown linears {unknown}")
    plan, route = [], None
    for path in paths:  # everything is checked before anything is replaced
        block, rel = blocks[known[path][0]], known[path][1]
        base = block.get_submodule(rel)
        if not isinstance(base, (nn.Linear, MXFP8Linear)):
            raise ValueError(f"{path} is a {type(base).__name__}, not a linear")
        device = base.weight_tiled.device if isinstance(base, MXFP8Linear) else base.weight.device
        route = route or AdapterRoute(names, device)
        stack = AdapterStack.of([adapters[n].get(path) for n in names], base.out_features, base.in_features, device)
        plan.append((block, rel, AdaptedLinear(base, stack, route)))
    for block, rel, module in plan:
        parent, _, leaf = rel.rpartition(".")
        setattr(block.get_submodule(parent), leaf, module)
    for block in blocks:
        attn = block.attn
        attn._adapter_qkv = _stacked_qkv((attn.to_q, attn.to_k, attn.to_v))
    transformer._qw_adapters = route
    return route


def remove_adapters(transformer):
    """Undo ``install_adapters``."""
    for block in transformer.transformer_blocks:
        for rel in LAYER_GROUPS["all"]:
            m = block.get_submodule(rel)
            if isinstance(m, AdaptedLinear):
                parent, _, leaf = rel.rpartition(".")
                setattr(block.get_submodule(parent), leaf, m.base)
        block.attn._adapter_qkv = None
    transformer._qw_adapters = None


__all__ = ["AdapterRoute", "AdapterStack", "AdaptedLinear", "running", "install_adapters", "remove_adapters"]
