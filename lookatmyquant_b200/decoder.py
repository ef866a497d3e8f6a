"""A Hugging Face causal model with its decoder layers' norms and residual additions on the kernels of `norms`.

The model's own forwards run around them and say what they do: `joined` gives a copy of the model that shares all of its modules,
with stand-ins for the decoder layers and the final norm, so that the masks, the positions, the multipliers of embeddings and
logits and the head are the model's. A stand-in runs its layer's own forward on symbols in the place of tensors. These record
which norm, which block (with the arguments that the layer gives it), which multiplier and which addition follow one another;
then the blocks run on tensors with `norms.norm` and `norms.join` between them. A layer that does anything else to a symbol
raises TypeError.
"""

from __future__ import annotations

import copy
import functools

import torch

from . import norms

_HOOKS = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")


def _refuse(what: str):
    raise TypeError(f"{what}: run_layers takes layers of RMS norms (a weight and a variance_epsilon), blocks and residual "
                    "additions")


def _passed_by(module):
    """Refuses a module whose own call the stand-ins leave out, where something hangs on that call."""
    if any(getattr(module, hooks) for hooks in _HOOKS):
        raise ValueError(f"run_layers passes by {type(module).__name__}, which has hooks")
    if "forward" in vars(module):
        _refuse(f"a forward put on one {type(module).__name__}")


class _Symbol:
    """In the place of a tensor in a layer's forward: what it is made from."""

    def __init__(self, kind, *of):
        self.kind, self.of = kind, of

    def __add__(self, other):
        return _Symbol("sum", self, other) if isinstance(other, _Symbol) else NotImplemented

    def __mul__(self, factor):
        return _Symbol("scaled", self, factor) if isinstance(factor, (int, float)) else NotImplemented

    __rmul__ = __mul__

    def __getitem__(self, k):
        if self.kind != "call" or k not in (0, 1):
            raise TypeError("not a block's tuple")
        return _Symbol("item", self, k)

    def __iter__(self):  # a block that returns its result and something beside it
        return iter((self[0], self[1]))


class _Child:
    """In the place of a layer's module while the layer runs on symbols."""

    def __init__(self, module):
        self.module = module

    def __call__(self, *args, **kwargs):
        if isinstance(self.module, torch.nn.Dropout):  # inactive: active ones are refused before
            return args[0]
        return _Symbol("call", self.module, args, kwargs)

    def __getattr__(self, name):
        return getattr(self.module, name)


class _Step:
    """stream + scale · post(block(... norm(stream) ...)[item])"""

    def __init__(self, norm, block, args, kwargs, taken, item, post, scale):
        self.norm, self.block, self.args, self.kwargs = norm, block, args, kwargs
        self.taken, self.item, self.post, self.scale = taken, item, post, scale

    def run(self, y):
        put = lambda x: y if x is self.taken else x
        out = self.block(*map(put, self.args), **{k: put(x) for k, x in self.kwargs.items()})
        if self.item is not None:
            out = out[self.item]
        if not isinstance(out, torch.Tensor):
            _refuse(f"what {type(self.block).__name__} returns")
        return out


@functools.cache
def _is_rms(cls, forward) -> bool:
    """Whether a module of this class with a weight w and a variance_epsilon is x · (mean(x²) + eps)^-1/2 · w: one is run."""
    try:
        module = cls.__new__(cls)
        torch.nn.Module.__init__(module)
        host = {"dtype": torch.float32, "device": "cpu"}
        x = torch.tensor([[1.0, -2.0, 0.5, 3.0], [0.25, 0.5, -0.125, 0.0625]], **host)
        w = torch.tensor([0.5, -2.0, 3.0, 1.25], **host)
        module.weight, module.variance_epsilon = torch.nn.Parameter(w, requires_grad=False), 0.25
        with torch.no_grad():
            got = forward(module, x)
            return torch.allclose(got, x * (x.square().mean(-1, keepdim=True) + 0.25).rsqrt() * w, rtol=1e-5, atol=0.0)
    except Exception:  # a norm that needs something else
        return False


def _is_norm(module) -> bool:
    return _is_rms(type(module), type(module).forward) and set(module._parameters) == {"weight"} and (
        isinstance(module.weight, torch.Tensor) and isinstance(module.variance_epsilon, float))


def _normed(x):
    """(the norm, its argument) where x is the result of a norm."""
    if isinstance(x, _Symbol) and x.kind == "call" and _is_norm(x.of[0]) and len(x.of[1]) == 1 and not x.of[2]:
        return x.of[0], x.of[1][0]
    return None, None


def _step(x, stream):
    """The step that adds x to the stream, or None."""
    scale, item = 1.0, None
    while x.kind == "scaled":
        x, scale = x.of[0], scale * x.of[1]
    post, arg = _normed(x)
    if post is not None:
        x = arg
    if isinstance(x, _Symbol) and x.kind == "item":
        x, item = x.of
    if not isinstance(x, _Symbol) or x.kind != "call":
        return None
    block, args, kwargs = x.of
    symbols = [a for a in (*args, *kwargs.values()) if isinstance(a, _Symbol)]
    if len(symbols) != 1:
        return None
    norm, of = _normed(symbols[0])
    return _Step(norm, block, args, kwargs, symbols[0], item, post, scale) if norm is not None and of is stream else None


def _steps(layer, args, kwargs) -> list:
    """What the layer's forward does with the stream, called with these arguments behind it."""
    name = type(layer).__name__
    _passed_by(layer)
    for child in layer.children():
        if isinstance(child, torch.nn.Dropout):
            _passed_by(child)
            if child.training and child.p:
                raise ValueError(f"run_layers: {name} drops elements of a block's result")
    symbolic = copy.copy(layer)
    symbolic.__dict__["_modules"] = {k: _Child(m) for k, m in layer._modules.items()}
    start = _Symbol("stream")
    try:
        out = symbolic.forward(start, *args, **kwargs)
    except Exception as e:
        raise TypeError(f"run_layers cannot follow {name}: its forward does more than norms, blocks and residual additions"
                        ) from e
    steps = []
    while out is not start:
        if not isinstance(out, _Symbol) or out.kind != "sum":
            _refuse(name)
        a, b = out.of
        step, out = _step(b, a), a
        if step is None:
            step, out = _step(a, b), b
        if step is None:
            _refuse(name)
        steps.append(step)
    for step in steps:
        for norm in (step.norm, step.post):
            if norm is not None:
                _passed_by(norm)
    return steps[::-1]


class _Stream:
    """The residual stream h, and the branch that is added to it with the next norm."""

    def __init__(self, h):
        self.h, self.branch, self.step = h, None, None

    def __getattr__(self, name):
        _refuse(f"a model that reads {name} of the states between its layers")

    def __getitem__(self, k):
        _refuse("a model that takes its layers' results apart")

    def normed(self, norm):
        """norm(h), the branch added to h before."""
        eps = norm.variance_epsilon
        if self.branch is None:
            return norms.norm(self.h, norm.weight, eps)
        branch, post = self.branch, self.step.post
        if post is not None and post.variance_epsilon != eps:  # a join has one eps
            branch, post = norms.norm(branch, post.weight, post.variance_epsilon), None
        self.h, y = norms.join(self.h, branch, norm.weight, post_weight=None if post is None else post.weight,
                               scale=self.step.scale, eps=eps)
        self.branch = None
        return y


class _Layer:
    """In the place of a decoder layer in the model's forward."""

    def __init__(self, layer):
        self._layer = layer

    def __getattr__(self, name):
        return getattr(self._layer, name)

    def __call__(self, hidden_states, *args, **kwargs):
        stream = hidden_states if isinstance(hidden_states, _Stream) else _Stream(hidden_states)
        for step in _steps(self._layer, args, kwargs):
            y = stream.normed(step.norm)
            stream.branch, stream.step = step.run(y), step
        return stream


class _Last:
    """In the place of the final norm."""

    def __init__(self, norm):
        self._norm = norm

    def __call__(self, x):
        return (x if isinstance(x, _Stream) else _Stream(x)).normed(self._norm)


def joined(model):
    """A copy of a Hugging Face causal model (model.model.layers, model.model.norm) that shares its modules and parameters and
    whose forward runs its decoder layers' norms and residual additions through `norms`: every addition goes into a join with
    the norm behind it, across the layers too. For one forward: what is set on the model later is not seen. No cache."""
    inner = getattr(model, "model", None)
    layers, norm = getattr(inner, "layers", None), getattr(inner, "norm", None)
    if not isinstance(layers, torch.nn.ModuleList) or not isinstance(norm, torch.nn.Module):
        _refuse(f"{type(model).__name__} without model.layers and model.norm")
    if not _is_norm(norm):
        _refuse(type(norm).__name__)
    _passed_by(norm)
    if any(getattr(m, "gradient_checkpointing", False) and m.training for m in (inner, *layers)):
        raise ValueError("run_layers keeps all states: gradient checkpointing is on")
    inside, outside = copy.copy(inner), copy.copy(model)
    inside.__dict__["_modules"] = {k: m for k, m in inner._modules.items() if k not in ("layers", "norm")}
    inside.__dict__["layers"], inside.__dict__["norm"] = [_Layer(layer) for layer in layers], _Last(norm)
    outside.__dict__["_modules"] = {**model._modules, "model": inside}
    return outside
