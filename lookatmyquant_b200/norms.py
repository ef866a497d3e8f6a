"""The norms around a model's blocks, joined with the residual addition, on B200 (liblamq_b200: lamq_norm_forward,
lamq_norm_backward).

A fine-tuning step around coded matrices runs a norm before every block and adds the block's result to the residual stream
behind it. `norm` is N(x; w) = x · (mean(x²) + eps)^-1/2 · (offset + w) over the last axis; `join` is a block's end and the next
one's beginning in one pass:

    p = N(branch; post_weight), or branch
    h = residual + scale · gate ⊙ p
    y = N(h; weight)

`norm_forward`, `norm_backward`, `join_forward` and `join_backward` are the same without autograd. A gate has the branch's shape
but for trailing axes of one before the last: (d,) for all rows, (batch, 1, d) for each text, (batch, length, d) for each
element. Tensors are fp32 or bf16: the norm's input and output share a type; the residual and h share one, branch and y one (an
fp32 stream takes bf16 branches, not the other way round); weights and the gate have types of their own. Sums are fp32 and
results are rounded once: y comes from h before its rounding. Rows have up to 16384 elements; inputs may be strided views
with a contiguous last axis (the norm's also the heads of a projection's output), outputs are contiguous. eps is positive.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import NORM_ARGS, check, launch_on, ptr

_DTYPES = {torch.float32: _lib.LAMQ_F32, torch.bfloat16: _lib.LAMQ_BF16}
_NONE = (0, 1, 0, 0)  # the lamq_rows of no tensor
_FAR = 1 << 29  # elements between the rows of a join that the library does not take
PARAMETERS = ("weight", "post_weight", "gate")


def _code(x: torch.Tensor, what: str) -> int:
    code = _DTYPES.get(x.dtype)
    if code is None or not x.is_cuda:
        raise TypeError(f"{what} must be a float32 or bfloat16 CUDA tensor")
    return code


def _rows(x: torch.Tensor, strides: int = 1):
    """(x, the lamq_rows of its rows), x copied where its rows do not lie at `strides` strides (one or two)."""
    d = x.shape[-1]
    if x.is_contiguous():
        return x, (x.data_ptr(), 1 << 30, d, 0)
    if x.stride(-1) == 1 or d == 1:
        axes = []  # (entries, stride), neighbours merged where they make one axis
        for n, s in zip(x.shape[:-1], x.stride()[:-1]):
            if n == 1:
                continue
            if axes and axes[-1][1] == n * s:
                axes[-1] = (axes[-1][0] * n, s)
            else:
                axes.append((n, s))
        if len(axes) <= 1 and (strides == 2 or not axes or axes[0][1] < _FAR):
            return x, (x.data_ptr(), 1 << 30, axes[0][1] if axes else d, 0)
        if len(axes) == 2 and strides == 2:
            return x, (x.data_ptr(), axes[1][0], axes[1][1], axes[0][1])
    x = x.contiguous()
    return x, (x.data_ptr(), 1 << 30, d, 0)


def _parameter(w: torch.Tensor | None, what: str, d: int, device):
    """(w, its type), contiguous."""
    if w is None:
        return None, 0
    code = _code(w, what)
    if w.shape != (d,) or w.device != device:
        raise ValueError(f"{what} must be a vector of {d} elements on {device}")
    return w if w.is_contiguous() else w.contiguous(), code


def _gate(gate: torch.Tensor | None, branch: torch.Tensor):
    """(gate, its type, how many of the branch's rows share a row of it)."""
    if gate is None:
        return None, 0, 1
    code = _code(gate, "the gate")
    shape = (1,) * (branch.ndim - gate.ndim) + tuple(gate.shape)
    same = 0
    while same < branch.ndim - 1 and shape[same] == branch.shape[same]:
        same += 1
    span = branch.shape[same:-1].numel()
    if len(shape) != branch.ndim or shape[-1] != branch.shape[-1] or any(n != 1 for n in shape[same:-1]) or (
            gate.device != branch.device):
        raise ValueError(f"the gate {tuple(gate.shape)} must have the branch's shape {tuple(branch.shape)} but for axes of one "
                         f"before the last, on {branch.device}")
    return gate if gate.is_contiguous() else gate.contiguous(), code, span


def _empty(like: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A contiguous tensor of `like`'s shape and device (empty_like without arguments takes half of torch.empty's 3 us)."""
    if like.dtype is dtype and like.is_contiguous():
        return torch.empty_like(like)
    return torch.empty_like(like, dtype=dtype, memory_format=torch.contiguous_format)


def _like(x: torch.Tensor, other: torch.Tensor, what: str, dtype=None):
    if x.shape != other.shape or x.device != other.device:
        raise ValueError(f"{what} {tuple(x.shape)} on {x.device} does not belong to {tuple(other.shape)} on {other.device}")
    if dtype is not None and x.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}, not {x.dtype}")



def norm_forward(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, offset: float = 0.0) -> torch.Tensor:
    """N(x; weight) over the last axis, of x's type and shape. x is read in place where its rows lie at one or two
    strides."""
    code = _code(x, "x")
    if x.ndim < 1:
        raise ValueError("x has no axis to norm over")
    d, dev = x.shape[-1], x.device
    weight, wcode = _parameter(weight, "the weight", d, dev)
    y = _empty(x, x.dtype)
    n = y.numel() // d if d else 0
    if not n:
        return y
    x, xr = _rows(x, 2)
    args = NORM_ARGS.pack(n, 1, d, code, code, wcode, 0, 0, 1.0, eps, offset, 0, *xr, *_NONE, weight.data_ptr(), 0, 0, 0,
                          y.data_ptr(), *_NONE, *_NONE, 0, 0, 0, 0, 0)
    here, stream = launch_on(dev)
    with here:
        check(_lib.load().lamq_norm_forward(args, stream), "lamq_norm_forward")
    return y


def _backward(n, args, dev, sums):
    lib = _lib.load()
    size = lib.lamq_norm_backward_workspace_size(args) if sums else 0
    ws = torch.empty_strided((size,), (1,), dtype=torch.uint8, device=dev) if size else None
    here, stream = launch_on(dev)
    with here:
        check(lib.lamq_norm_backward(args, ptr(ws), size, stream), "lamq_norm_backward")


def norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, offset: float = 0.0,
                  want=PARAMETERS):
    """(dx, dweight) of `norm_forward` for the result's gradient dy; dweight is None unless "weight" is in `want`. Equal
    calls give equal bits."""
    code = _code(x, "x")
    if x.ndim < 1:
        raise ValueError("x has no axis to norm over")
    _like(dy, x, "dy", x.dtype)
    d, dev = x.shape[-1], x.device
    weight, wcode = _parameter(weight, "the weight", d, dev)
    dx = _empty(x, x.dtype)
    n = dx.numel() // d if d else 0
    dw = None
    if "weight" in want:
        dw = torch.empty_like(weight)
    if not n:
        return dx, None if dw is None else dw.zero_()
    x, xr = _rows(x, 2)
    dy, dyr = _rows(dy, 2)
    args = NORM_ARGS.pack(n, 1, d, code, code, wcode, 0, 0, 1.0, eps, offset, 0, *xr, *_NONE, weight.data_ptr(), 0, 0, 0, 0,
                          *_NONE, *dyr, dx.data_ptr(), 0, ptr(dw) or 0, 0, 0)
    _backward(n, args, dev, dw is not None)
    return dx, dw


def _join_types(residual, branch):
    if branch.ndim < 1:
        raise ValueError("the branch has no axis to norm over")
    _like(branch, residual, "the branch")
    rcode, bcode = _code(residual, "the residual"), _code(branch, "the branch")
    if rcode != bcode and rcode != _lib.LAMQ_F32:
        raise TypeError("a bfloat16 residual takes a bfloat16 branch")
    return rcode, bcode


def join_forward(residual: torch.Tensor, branch: torch.Tensor, weight: torch.Tensor | None = None,
                 post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float = 1.0,
                 eps: float = 1e-6, offset: float = 0.0):
    """(h, y) with h = residual + scale · gate ⊙ N(branch; post_weight) in the residual's type and y = N(h; weight) in the
    branch's; without a post_weight the branch goes in as it is, without a gate its factor is 1, without a weight y is
    None."""
    rcode, bcode = _join_types(residual, branch)
    d, dev = branch.shape[-1], branch.device
    weight, wcode = _parameter(weight, "the weight", d, dev)
    post, pcode = _parameter(post_weight, "the post_weight", d, dev)
    gate, gcode, span = _gate(gate, branch)
    h = _empty(branch, residual.dtype)
    y = None if weight is None else _empty(branch, branch.dtype)
    n = h.numel() // d if d else 0
    if not n:
        return h, y
    residual, rr = _rows(residual)
    branch, br = _rows(branch)
    args = NORM_ARGS.pack(n, span, d, rcode, bcode, wcode, pcode, gcode, scale, eps, offset, 0, *rr, *br, ptr(weight) or 0,
                          ptr(post) or 0, ptr(gate) or 0, h.data_ptr(), ptr(y) or 0, *_NONE, *_NONE, 0, 0, 0, 0, 0)
    here, stream = launch_on(dev)
    with here:
        check(_lib.load().lamq_norm_forward(args, stream), "lamq_norm_forward")
    return h, y


def join_backward(dh: torch.Tensor | None, dy: torch.Tensor | None, h: torch.Tensor, branch: torch.Tensor,
                  weight: torch.Tensor | None = None, post_weight: torch.Tensor | None = None,
                  gate: torch.Tensor | None = None, scale: float = 1.0, eps: float = 1e-6, offset: float = 0.0,
                  want=PARAMETERS):
    """(d_residual, d_branch, d_weight, d_post_weight, d_gate) of `join_forward` for the gradients dh of h and dy of y (None:
    zero), with the h that it returned. What the call had no tensor for, or `want` does not name, is None. Where the branch
    enters h unchanged (no post_weight, no gate, scale 1, one type) its gradient is the residual's: the same tensor is
    returned twice. Equal calls give equal bits."""
    rcode, bcode = _join_types(h, branch)
    d, dev = branch.shape[-1], branch.device
    weight, wcode = _parameter(weight, "the weight", d, dev)
    post, pcode = _parameter(post_weight, "the post_weight", d, dev)
    gate, gcode, span = _gate(gate, branch)
    if dh is not None:
        _like(dh, h, "dh", h.dtype)
    if dy is not None:
        if weight is None:
            raise ValueError("dy belongs to a weight")
        _like(dy, branch, "dy", branch.dtype)
    dr = _empty(branch, h.dtype)
    same = post is None and gate is None and scale == 1.0 and rcode == bcode
    db = dr if same else _empty(branch, branch.dtype)
    dw = None if weight is None or "weight" not in want else torch.empty_like(weight)
    du = None if post is None or "post_weight" not in want else torch.empty_like(post)
    dg = None if gate is None or "gate" not in want else torch.empty_like(gate)
    n = dr.numel() // d if d else 0
    if not n:
        return dr, db, *(None if x is None else x.zero_() for x in (dw, du, dg))
    h, hr = _rows(h)
    branch, br = _rows(branch)
    dh, dhr = (None, _NONE) if dh is None else _rows(dh)
    dy, dyr = (None, _NONE) if dy is None else _rows(dy)
    args = NORM_ARGS.pack(n, span, d, rcode, bcode, wcode, pcode, gcode, scale, eps, offset, 0, *hr, *br, ptr(weight) or 0,
                          ptr(post) or 0, ptr(gate) or 0, 0, 0, *dhr, *dyr, dr.data_ptr(), 0 if same else db.data_ptr(),
                          ptr(dw) or 0, ptr(du) or 0, ptr(dg) or 0)
    _backward(n, args, dev, dw is not None or du is not None or dg is not None)
    return dr, db, dw, du, dg


class _Once(torch.autograd.Function):
    """Gradients that come from kernels which leave no graph behind, made to depend on what they were computed from:
    differentiating them raises."""

    @staticmethod
    def forward(ctx, count, *tensors):
        return tuple(None if g is None else g.view_as(g) for g in tensors[-count:])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("the lamq norms have no second derivatives")


def _once(grads, *sources):
    return _Once.apply(len(grads), *sources, *grads) if torch.is_grad_enabled() else grads  # enabled: create_graph


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, offset):
        ctx.save_for_backward(x, weight)
        ctx.rest = (eps, offset)
        return norm_forward(x, weight, eps, offset)

    @staticmethod
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        grads = norm_backward(dy, x, weight, *ctx.rest, want=PARAMETERS[:1] if ctx.needs_input_grad[1] else ())
        return (*_once(grads, dy, x, weight), None, None)


class _Join(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, branch, weight, post_weight, gate, scale, eps, offset):
        h, y = join_forward(residual, branch, weight, post_weight, gate, scale, eps, offset)
        ctx.save_for_backward(h, branch, weight, post_weight, gate)
        ctx.rest = (scale, eps, offset)
        ctx.set_materialize_grads(False)
        return h, y

    @staticmethod
    def backward(ctx, dh, dy):
        if dh is None and dy is None:
            return (None,) * 8
        h, branch, weight, post, gate = ctx.saved_tensors
        want = [name for name, needed in zip(PARAMETERS, ctx.needs_input_grad[2:5]) if needed]
        grads = join_backward(dh, dy, h, branch, weight, post, gate, *ctx.rest, want=want)
        return (*_once(grads, dh, dy, h, branch, weight, post, gate), None, None, None)


def norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, offset: float = 0.0) -> torch.Tensor:
    """`norm_forward` under autograd: its gradients are `norm_backward`'s (once: differentiating them raises)."""
    return _Norm.apply(x, weight, eps, offset)


def join(residual: torch.Tensor, branch: torch.Tensor, weight: torch.Tensor | None = None,
         post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float = 1.0, eps: float = 1e-6,
         offset: float = 0.0):
    """`join_forward`'s (h, y) under autograd: its gradients are `join_backward`'s (once: differentiating them raises)."""
    return _Join.apply(residual, branch, weight, post_weight, gate, scale, eps, offset)


def run_layers(model, x: torch.Tensor) -> torch.Tensor:
    """What model.model(inputs_embeds=x) gives behind its final norm, for a Hugging Face causal model and the embedded whole
    windows x (batch, length, d): the model's own masks, positions, attention and MLP modules, and `norm` and `join` in the
    place of its decoder layers' norms and residual additions, each of which goes into the join with the norm behind it, across
    the layers too (a layer's norms behind its blocks and a multiplier of their results included). Layers that do anything else, and
    other norms than x · (mean(x²) + eps)^-1/2 · w, raise TypeError; hooks on the layers and norms that are not called, active
    dropout between them and gradient checkpointing raise ValueError. No cache and no padding."""
    from .decoder import joined  # it calls this module
    return joined(model).model(inputs_embeds=x, use_cache=False).last_hidden_state
