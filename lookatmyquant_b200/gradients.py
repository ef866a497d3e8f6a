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


def _device(tensors):
    for x in tensors:
        if isinstance(x, torch.Tensor):
            return x.device
        if x is not None:
            _refuse(x, None, "gradients")
    raise ValueError("no gradients")


def _refuse(x, device, what):
    if not isinstance(x, torch.Tensor) or x.layout is not torch.strided or x.dtype not in _DTYPES or not x.is_cuda:
        raise TypeError(f"{what} must be dense float32 or bfloat16 CUDA tensors")
    raise ValueError(f"{what} on {x.device} and {device}: one call takes those of one device")


def _code(x, index, device, what) -> int:
    """The type of a tensor on `device` (whose index is given), which is refused if it is none of this module's. (A few
    attributes of every tensor: 0.3 us each is half of what a list costs the host.)"""
    code = _DTYPES.get(x.dtype) if isinstance(x, torch.Tensor) else None
    if code is None or x.layout is not torch.strided or x.get_device() != index:
        _refuse(x, device, what)
    return code


def _call(name, values, count, device, *rest):
    """A C call over `count` tensors, whose `values` are (pointer, pointer of the output, elements, type, type of the output)
    one behind the other. The norm."""
    lib = _lib.load()
    table = struct.pack("=" + _lib.GRADIENT.format[1:] * count, *values)
    norm = torch.empty_strided((), (), dtype=torch.float32, device=device)
    size = lib.lamq_gradient_workspace_size(count)
    ws = torch.empty_strided((size,), (1,), dtype=torch.uint8, device=device)
    here, stream = launch_on(device)
    with here:
        check(getattr(lib, name)(table, count, *rest, norm.data_ptr(), ws.data_ptr(), size, stream), name)
    return norm


def global_norm(tensors) -> torch.Tensor:
    """The square root of the sum of squares over all `tensors` (fp32 or bf16, None entries are left out) as an fp32 scalar
    on their device. Squares that fp32 would lose or overflow are summed in fp64. Equal calls give equal bits."""
    tensors = list(tensors)
    device = _device(tensors)
    index, values, count, copies = device.index if device.type == "cuda" else -2, [], 0, []
    for x in tensors:
        if x is None:
            continue
        code = _code(x, index, device, "gradients")
        if not x.is_contiguous() and not _dense(x):
            x = x.contiguous()
            copies.append(x)  # alive until the launch
        values += (x.data_ptr(), 0, x.numel(), code, 0)
        count += 1
    return _call("lamq_gradient_norm", values, count, device)


def clip(tensors, max_norm: float, out=None, eps: float = 1e-6) -> torch.Tensor:
    """Scales `tensors` by min(1, max_norm / (norm + eps)), norm their `global_norm`, which is returned. In place, and then
    untouched where the norm is within the bound; or, with `out`, into its tensors (one for each, of its shape, fp32 or bf16).
    A norm that is NaN makes everything NaN, an infinite one zeros (infinite elements NaN), as in torch. Tensors that share
    memory raise ValueError: they would be scaled twice (views with gaps, which go through copies, only where two are the
    same)."""
    tensors = list(tensors)
    into = tensors if out is None else list(out)
    if len(into) != len(tensors):
        raise ValueError(f"{len(into)} outputs for {len(tensors)} gradients")
    device = _device(tensors)
    index, values, count, copies = device.index if device.type == "cuda" else -2, [], 0, []
    late, written, gaps = [], [], set()  # (tensor, what is copied into it afterwards); what changes; the views with gaps
    for x, o in zip(tensors, into):
        if x is None:
            continue
        code = to = _code(x, index, device, "gradients")
        written.append(o)
        if o is not x:
            to = _code(o, index, device, "outputs")
            if o.shape != x.shape:
                raise ValueError(f"an output {tuple(o.shape)} for a gradient {tuple(x.shape)}")
        if not o.is_contiguous() and not _dense(o):
            place = (o.data_ptr(), o.shape, o.stride())
            if place in gaps or any(n != 1 and step == 0 for n, step in zip(o.shape, o.stride())):
                raise ValueError("tensors of the list overlap where they are written")
            gaps.add(place)
            copies.append(x.contiguous())  # alive until the launch
            late.append((o, copies[-1] if o is x else torch.empty(o.shape, dtype=o.dtype, device=device)))
            x, o = copies[-1], late[-1][1]
        elif o is not x and not (x.is_contiguous() and o.is_contiguous()) and not (_dense(x) and x.stride() == o.stride()):
            x = torch.empty_strided(o.shape, o.stride(), dtype=x.dtype, device=device).copy_(x.detach())
            copies.append(x)
        values += (x.data_ptr(), o.data_ptr(), x.numel(), code, to)
        count += 1
    norm = _call("lamq_gradient_clip", values, count, device, float(max_norm), float(eps))
    torch.autograd.graph.increment_version([o for o in written if not o.is_inference()])
    for o, value in late:
        with torch.inference_mode() if o.is_inference() else torch.no_grad():
            o.copy_(value)
    return norm
