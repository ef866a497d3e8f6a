"""The global norm of many gradients, and their clipping, on B200 (liblamq_b200: lamq_gradient_norm, lamq_gradient_clip).

What a training step does between its backward pass and its update: the Euclidean norm over all gradients together, and all of
them scaled down where it is above a bound. A list of any number of fp32 and bf16 tensors on one device goes in two launches
for every thousand of them; the norm stays on the device, so nothing waits for it.
"""

from __future__ import annotations

import struct

import torch

from . import _lib
from ._lib import check, launch_on

_DTYPES = {torch.float32: _lib.LAMQ_F32, torch.bfloat16: _lib.LAMQ_BF16}


def _dense(x: torch.Tensor) -> bool:
    """Whether the elements fill one piece of memory, in whatever order of the axes."""
    if x.is_contiguous():
        return True
    step = 1
    for s, n in sorted((s, n) for n, s in zip(x.shape, x.stride()) if n != 1):
        if s != step:
            return False
        step *= n
    return True


def _check(x, device, what="gradients"):
    if not isinstance(x, torch.Tensor) or x.layout is not torch.strided or x.dtype not in _DTYPES or not x.is_cuda:
        raise TypeError(f"{what} must be dense float32 or bfloat16 CUDA tensors")
    if x.device != device:
        raise ValueError(f"{what} on {x.device} and {device}: one call takes those of one device")


def _call(name, items, device, *rest):
    """A C call over `items`, (pointer, pointer of the output, elements, type, type of the output) each. The norm."""
    lib = _lib.load()
    table = struct.pack("=" + "2Qq2i" * len(items), *(x for item in items for x in item))
    norm = torch.empty((), dtype=torch.float32, device=device)
    size = lib.lamq_gradient_workspace_size(len(items))
    ws = torch.empty(size, dtype=torch.uint8, device=device)
    here, stream = launch_on(device)
    with here:
        check(getattr(lib, name)(table, len(items), *rest, norm.data_ptr(), ws.data_ptr(), size, stream), name)
    return norm


def _listed(tensors):
    tensors = [x for x in tensors if x is not None]
    if not tensors:
        raise ValueError("no gradients")
    device = getattr(tensors[0], "device", None)
    for x in tensors:
        _check(x, device)
    return tensors, device


def global_norm(tensors) -> torch.Tensor:
    """The square root of the sum of squares over all `tensors` (fp32 or bf16, None entries are left out) as an fp32 scalar
    on their device. Squares that fp32 would lose or overflow are summed in fp64. Equal calls give equal bits."""
    tensors, device = _listed(tensors)
    tensors = [x if _dense(x) else x.contiguous() for x in tensors]
    return _call("lamq_gradient_norm", [(x.data_ptr(), 0, x.numel(), _DTYPES[x.dtype], 0) for x in tensors], device)


def clip(tensors, max_norm: float, out=None, eps: float = 1e-6) -> torch.Tensor:
    """Scales `tensors` by min(1, max_norm / (norm + eps)), norm their `global_norm`, which is returned. In place, and then
    untouched where the norm is within the bound; or, with `out`, into its tensors (one for each, of its shape, fp32 or bf16).
    A norm that is NaN makes everything NaN, an infinite one zeros (infinite elements NaN), as in torch. Tensors that share
    memory raise ValueError: they would be scaled twice."""
    tensors = list(tensors)
    into = tensors if out is None else list(out)
    if len(into) != len(tensors):
        raise ValueError(f"{len(into)} outputs for {len(tensors)} gradients")
    pairs = [(x, o) for x, o in zip(tensors, into) if x is not None]
    tensors, device = _listed(x for x, _ in pairs)
    items, late, written = [], [], []
    for x, o in pairs:
        if o is not x:
            _check(o, device, "outputs")
            if o.shape != x.shape:
                raise ValueError(f"an output {tuple(o.shape)} for a gradient {tuple(x.shape)}")
        written.append(o)
        if o is x:
            if not _dense(x):
                x = x.contiguous()
                late.append((o, x))
            o = x
        elif not (x.is_contiguous() and o.is_contiguous()) and not (_dense(x) and x.stride() == o.stride()):
            x = x.contiguous()
            if not o.is_contiguous():
                late.append((o, torch.empty(o.shape, dtype=o.dtype, device=device)))
                o = late[-1][1]
        items.append((x, o))  # keeps copies until the launch
    norm = _call("lamq_gradient_clip", [(x.data_ptr(), o.data_ptr(), x.numel(), _DTYPES[x.dtype], _DTYPES[o.dtype])
                                        for x, o in items], device, float(max_norm), float(eps))
    torch.autograd.graph.increment_version(written)
    for o, value in late:
        with torch.no_grad():
            o.copy_(value)
    return norm
