"""Attention for training steps on B200 (liblamq_b200: lamq_attention_forward, lamq_attention_backward).

The model passes this package runs gradients through (importance.row_importance, importance.guided_weights, and a
fine-tuning step around trellis-coded matrices) spend their attention here: `forward` keeps, beside the output, one
number per query (lse, the logarithm of the sum of exponentials); `backward` recomputes the probabilities from it, so
that nothing of size queries x keys is ever stored. `attention` is the two under autograd, and `use_in_transformers`
makes it an attention implementation of Hugging Face models ("lamq").

Tensors are (batch, heads, length, head_dim) bf16 views with contiguous head_dim (a projection's (batch, length, heads,
head_dim) output transposed is read in place); outputs come in that memory order too. Heads may be shared: query head h
reads key head h // (heads // kv_heads). Query i of text b sees keys key_start[b] <= j < key_end[b] and, when causal,
j <= i + kv_len - q_len. A query that sees no key gives a zero output, lse -inf and no gradient. head_dim is a multiple of
8 up to 128, the scale positive and finite; anything else raises ValueError.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import ATTENTION_ARGS, check, launch_on, ptr

_STATUS = _lib.StatusWord("attention")


def check_status():
    """Raises if a kernel of any call so far gave up on a device wait (its results are then invalid). Waits for the
    device."""
    _STATUS.check()


def _heads(x: torch.Tensor, what: str):
    """(x, what lamq_heads holds of it), x copied where TMA cannot read it in place."""
    if x.dtype is not torch.bfloat16 or not x.is_cuda:
        raise TypeError(f"{what} must be a bfloat16 CUDA tensor")
    if x.ndim != 4:
        raise ValueError(f"{what} must be (batch, heads, length, head_dim)")
    b, h, r, one = x.stride()
    p = x.data_ptr()
    if one != 1 or (b | h | r) & 7 or p & 15 or b <= 0 or h <= 0 or r <= 0:
        n, m, k, d = x.shape  # the stride of an axis of one entry does not matter
        if d and ((one != 1 and d > 1) or p & 15 or (n > 1 and (b & 7 or b <= 0)) or (m > 1 and (h & 7 or h <= 0)) or
                  (k > 1 and (r & 7 or r <= 0))):
            y = x.contiguous()
            x = y if y.data_ptr() & 15 == 0 else y.clone()  # a contiguous tensor may start between two 16-byte pieces
            b, h, r, one = x.stride()
            p = x.data_ptr()
    return x, (p, b, h, r)


def _like_projection(B: int, H: int, L: int, D: int, device):
    """An empty (B, H, L, D) tensor in the memory order of a projection's (B, L, H·D) output, as _heads gives it."""
    strides = (L * H * D, D, H * D)
    x = torch.empty_strided((B, H, L, D), (*strides, 1), dtype=torch.bfloat16, device=device)
    return x, (x.data_ptr(), *strides)


def _bounds(x: torch.Tensor | None, what: str, batch: int, device):
    if x is None:
        return None
    if x.dtype != torch.int32 or x.device != device or x.shape != (batch,):
        raise ValueError(f"{what} must be an int32 tensor of {batch} entries on {device}")
    return x.contiguous()


def _shapes(q, k, v, scale):
    B, Hq, Lq, D = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    shape = (B, Hkv, Lk, D)
    if k.shape != shape or v.shape != shape or k.device != q.device or v.device != q.device:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    return B, Hq, Hkv, D, Lq, Lk, D ** -0.5 if scale is None else float(scale)


def forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float | None = None, causal: bool = True,
            key_start: torch.Tensor | None = None, key_end: torch.Tensor | None = None):
    """softmax(scale·q·kᵀ)·v over each query's keys (scale: head_dim^-1/2 by default): (output, lse), the output bf16
    like q and lse (batch, heads, q length) fp32."""
    (q, qh), (k, kh), (v, vh) = _heads(q, "q"), _heads(k, "k"), _heads(v, "v")
    B, Hq, Hkv, D, Lq, Lk, scale = _shapes(q, k, v, scale)
    dev = q.device
    start, end = _bounds(key_start, "key_start", B, dev), _bounds(key_end, "key_end", B, dev)
    o, oh = _like_projection(B, Hq, Lq, D, dev)
    lse = torch.empty((B, Hq, Lq), dtype=torch.float32, device=dev)
    args = ATTENTION_ARGS.pack(B, Hq, Hkv, D, causal, Lq, Lk, scale, 0, ptr(start) or 0, ptr(end) or 0, *qh, *kh, *vh,
                               *oh, lse.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    here, stream = launch_on(dev)
    with here:
        check(_lib.load().lamq_attention_forward(args, _STATUS.on(dev).data_ptr(), stream), "lamq_attention_forward")
    return o, lse


def backward(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
             scale: float | None = None, causal: bool = True, key_start: torch.Tensor | None = None,
             key_end: torch.Tensor | None = None):
    """(dq, dk, dv) of `forward` for the output's gradient `do`, with the o and lse that `forward` returned for the
    same q, k, v, scale, causal and key ranges. Equal calls give equal bits."""
    (q, qh), (k, kh), (v, vh) = _heads(q, "q"), _heads(k, "k"), _heads(v, "v")
    (o, oh), (do, doh) = _heads(o, "o"), _heads(do, "do")
    B, Hq, Hkv, D, Lq, Lk, scale = _shapes(q, k, v, scale)
    dev = q.device
    if o.shape != q.shape or do.shape != q.shape or o.device != dev or do.device != dev:
        raise ValueError(f"o {tuple(o.shape)} and do {tuple(do.shape)} must be like q {tuple(q.shape)}")
    if lse.shape != (B, Hq, Lq) or lse.dtype is not torch.float32 or lse.device != dev:
        raise ValueError(f"lse must be a float32 tensor of shape {(B, Hq, Lq)}")
    lse = lse.contiguous()
    start, end = _bounds(key_start, "key_start", B, dev), _bounds(key_end, "key_end", B, dev)
    dq, dqh = _like_projection(B, Hq, Lq, D, dev)
    dk, dkh = _like_projection(B, Hkv, Lk, D, dev)
    dv, dvh = _like_projection(B, Hkv, Lk, D, dev)
    if Hq == 0:  # nothing reads the keys, and the library has nothing to run
        return dq, dk.zero_(), dv.zero_()
    lib = _lib.load()
    size = lib.lamq_attention_backward_workspace_size(B, Hq, Lq)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    args = ATTENTION_ARGS.pack(B, Hq, Hkv, D, causal, Lq, Lk, scale, 0, ptr(start) or 0, ptr(end) or 0, *qh, *kh, *vh,
                               *oh, lse.data_ptr(), *doh, *dqh, *dkh, *dvh)
    here, stream = launch_on(dev)
    with here:
        check(lib.lamq_attention_backward(args, ws.data_ptr(), size, _STATUS.on(dev).data_ptr(), stream),
              "lamq_attention_backward")
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, causal, key_start, key_end):
        o, lse = forward(q, k, v, scale, causal, key_start, key_end)
        ctx.save_for_backward(q, k, v, o, lse, key_start, key_end)
        ctx.scale, ctx.causal = scale, causal
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse, start, end = ctx.saved_tensors
        grads = backward(do, q, k, v, o, lse, ctx.scale, ctx.causal, start, end)
        if torch.is_grad_enabled():  # create_graph
            grads = _Once.apply(do, q, k, v, *grads)
        return (*grads, None, None, None, None)


class _Once(torch.autograd.Function):
    """The gradients, which come from kernels that leave no graph behind, made to depend on what they were computed from:
    differentiating them raises. (torch's once_differentiable lets them pass for constants where `do` is one.)"""

    @staticmethod
    def forward(ctx, do, q, k, v, *grads):
        return tuple(g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("the lamq attention has no second derivatives")


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float | None = None, causal: bool = True,
              key_start: torch.Tensor | None = None, key_end: torch.Tensor | None = None) -> torch.Tensor:
    """`forward`'s output under autograd: its gradients are `backward`'s (once: differentiating them raises)."""
    return _Attention.apply(q, k, v, scale, causal, key_start, key_end)


def _transformers_attention(module, query, key, value, attention_mask, scaling=None, dropout=0.0, **kwargs):
    for what in ("sliding_window", "softcap", "s_aux"):
        if kwargs.get(what) is not None:
            raise NotImplementedError(f"the lamq attention has no {what}")
    if attention_mask is not None or dropout:
        raise NotImplementedError("the lamq attention takes whole windows: no mask and no dropout")
    causal = kwargs.get("is_causal")
    causal = getattr(module, "is_causal", True) if causal is None else causal
    return attention(query, key, value, scaling, causal).transpose(1, 2), None


def _transformers_mask(batch_size, q_length, kv_length, q_offset=0, kv_offset=0, mask_function=None,
                       attention_mask=None, **kwargs):
    from transformers.masking_utils import causal_mask_function
    if mask_function not in (None, causal_mask_function) or kv_offset or int(q_offset) + q_length != kv_length or (
            attention_mask is not None and not bool(attention_mask.all())):
        raise NotImplementedError("the lamq attention takes whole windows: no padding, packing or windowed mask")
    return None


def use_in_transformers(name: str = "lamq") -> str:
    """Registers `attention` with Hugging Face transformers under `name` (returned): a model whose config has
    `_attn_implementation = name` runs its attention forwards and backwards on these kernels. bf16 models on whole
    windows: a padded, packed or windowed mask raises NotImplementedError."""
    from transformers import AttentionInterface, AttentionMaskInterface
    AttentionInterface.register(name, _transformers_attention)
    AttentionMaskInterface.register(name, _transformers_mask)
    return name
