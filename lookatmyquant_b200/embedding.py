"""Embedding tables by frequency buckets on B200: the host side of quantize.py's `embedding_buckets`,
`frequency_order`, `embed_word` and `quantize_embedding` (ShinMegamiBoson/lookatmyquant, quantize.py:350-365,
:395-465) for the trellis family and the bucket programs without a code.

A bucket of embedding rows is rotated over the hidden dimension only (each row stays its own, so a lookup decodes one
row), split into a 16-bit RMS scale per row, and coded with a column trellis over runs of 256 rows (TrellisCode with
T = 256: down each hidden column, 256 consecutive rows form one free-start path) — under block LDLQ with the table's
input statistics H, or by plain Viterbi rounding when H is None or the identity (a lookup table). Rows are padded with
zero rows to whole runs of 256 and dropped after. The compute runs in liblamq_b200.so: the rotation through the
Hadamard factors (lamq_rht_rows), the environment (lamq_env_factor), the column-trellis sweep (lamq_ldlq_coltrellis)
or the Viterbi (lamq_viterbi). `lm`/`ter` scalar-code buckets and sliced (per-layer-input) tables are not on this
path and raise NotImplementedError.

A training step's side of a table is here too: `lookup` (rows by token id, scaled), `lookup_gradient` (the table's
gradient, summed in the tokens' order: bit-reproducible) and `scaled_embedding`, the two under autograd.
"""

from __future__ import annotations

import torch

from . import _lib, codes
from ._lib import check, launch_on, ptr
from .quantize import Dense, parse
from .rotation import Rotation

EMBED_T = 256  # embedding rows per trellis run (quantize.py:99)


def embedding_buckets(V: int, first: int = 256) -> list:
    """Sizes of the buckets of a V-row table ranked by frequency (quantize.py:350-358): first, first, then doubling,
    the last bucket the rest."""
    sizes, s = [first], first
    while sum(sizes) + s < V:
        sizes.append(s)
        s *= 2
    return sizes + [V - sum(sizes)]


def frequency_order(ids: torch.Tensor, V: int) -> torch.Tensor:
    """Token ids by count in `ids`, most frequent first, ties by id (quantize.py:361-364)."""
    counts = torch.bincount(ids.reshape(-1).cpu(), minlength=V)[:V]
    return torch.sort(-counts, stable=True).indices


def embed_word(W: torch.Tensor, H: torch.Tensor | None, program: str, seed: int, center: bool = False,
               device=None):
    """One bucket of embedding rows (quantize.py:395-446): a Dense word (the dequantized rows, fp64 on the device, and
    the bits its format stores). Families: tr<b> (column trellis over runs of 256 rows, L = 12, the package's T = 256
    tables), fp16, mean, zero, prng; `center` stores the bucket's mean row apart (16 bits a value)."""
    dev = codes._dev(device)
    fam, b, _ = parse(program)
    W = W.to(dev)
    if center and fam not in ("fp", "mean", "prng", "zero"):
        m = W.double().mean(0, keepdim=True)
        q = embed_word(W.double() - m, H, program, seed, device=dev)
        return Dense(q.matrix() + m, q.rate_bits() + 16 * W.shape[1])
    if fam == "fp":
        return Dense(W.to(torch.bfloat16).double(), 16 * W.numel())
    if fam == "mean":
        return Dense(W.double().mean(0, keepdim=True).expand_as(W).clone(), 16 * W.shape[1])
    if fam == "zero":
        return Dense(torch.zeros_like(W, dtype=torch.float64), 0)
    if fam == "prng":  # what is stored: the mean row and each column's spread; the noise from torch's CPU generator
        m = W.double().mean(0, keepdim=True)
        noise = torch.randn(W.shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dev)
        return Dense(m + noise * (W.double() - m).std(0, keepdim=True), 32 * W.shape[1])
    if fam != "tr":
        raise NotImplementedError(f"embedding program family {fam!r} is outside the B200 hot path (trellis codes)")
    n = W.shape[1]
    lookup = H is None or bool(torch.equal(H.cpu().double(), torch.eye(len(H), dtype=torch.float64)))
    R = Rotation(n, seed, dev)
    rows = W.shape[0]
    pad = (-rows) % EMBED_T
    Wp = torch.cat([W.double(), torch.zeros(pad, n, dtype=torch.float64, device=dev)]) if pad else W.double()
    # the reference rotates in fp32 (a wide table is a large product); the values are rounded to fp32 as it does
    Wr = R.rows(Wp.float().double()).float().double()
    Hr = None if lookup else R.conj(H.to(dev, torch.float64))
    code = codes.TrellisCode(12, b, T=EMBED_T)
    net = codes.ldlq_words([Wr], Hr, code, [seed], incoherent=False, device=dev)[0]
    Q = net.matrix(dtype=torch.float64)[:rows]
    out = R.rows_t(Q.float().double()).float().double()
    return Dense(out, net.rate_bits() * rows / (rows + pad))


@torch.no_grad()
def quantize_embedding(E: torch.Tensor, spec: dict, H: torch.Tensor | None, order: torch.Tensor, seed0: int = 7000,
                       center: bool = False, seed_shift: int = 0):
    """One table, bucket by bucket as the plan says (quantize.py:449-465): spec = {"sizes": [...], "programs": [...]},
    `order` the rows by frequency. E is written in place with each bucket's dequantized rows; returns (bits, weights)."""
    bits, lo = 0.0, 0
    for k, (size, p) in enumerate(zip(spec["sizes"], spec["programs"])):
        rows = order[lo:lo + size].to(E.device)
        net = embed_word(E.data[rows].double(), H, p, seed0 + k + seed_shift, center=center, device=E.device)
        E.data[rows] = net.matrix(dtype=torch.float64).to(E.dtype).to(E.device)
        bits += net.rate_bits()
        lo += size
    return bits, E.numel()


_STATUS = _lib.StatusWord("embedding", "embedding ids outside the table")
_DTYPES = {torch.float32: _lib.LAMQ_F32, torch.bfloat16: _lib.LAMQ_BF16}


def check_status():
    """Raises ValueError if a lookup or gradient so far met an id outside its table (its row is taken as zero), and
    LamqError if a kernel gave up on a device wait (then no sums were written; reported
    before a bad id). Waits for the device."""
    _STATUS.check()


def _matrix(x: torch.Tensor, what: str):
    """(x, its leading dimension, its type in the C ABI), x copied where its rows are not contiguous."""
    code = _DTYPES.get(x.dtype)
    if code is None or not x.is_cuda:
        raise TypeError(f"{what} must be a float32 or bfloat16 CUDA tensor")
    ld, one = x.stride()
    rows, d = x.shape
    if one != 1 or ld < d:
        if (one != 1 and d > 1) or (ld < d and rows > 1):
            x = x.contiguous()
            ld = x.stride(0)
        ld = max(ld, d)  # of a single row or column: any
    return x, ld, code


def _rows_like(shape, d: int, x: torch.Tensor) -> torch.Tensor:
    """An empty contiguous tensor of shape + (d,), of x's type and device."""
    if len(shape) == 1:
        return torch.empty_strided((shape[0], d), (d, 1), dtype=x.dtype, device=x.device)
    return torch.empty((*shape, d), dtype=x.dtype, device=x.device)


def _ids(ids: torch.Tensor, device) -> torch.Tensor:
    if ids.dtype not in (torch.int64, torch.int32) or ids.device != device:
        raise TypeError("ids must be an int64 or int32 tensor on the table's device")
    return ids if ids.is_contiguous() else ids.contiguous()


def _padding(padding_idx: int | None, rows: int) -> int:
    """The row, or -1 for none; negative indices count from the table's end, as in torch."""
    if padding_idx is None:
        return -1
    if not -rows <= padding_idx < rows:
        raise ValueError(f"padding_idx {padding_idx} outside the table's {rows} rows")
    return padding_idx % rows


def lookup(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    """scale · table[ids] (ids of any shape; table V x d fp32 or bf16; the result in the table's type, the product in
    fp32). Tokens with id `padding_idx` get zero rows, whatever the table holds there. An id outside the table gets a zero
    row and is reported by `check_status()`."""
    if table.ndim != 2:
        raise ValueError("the table must be a matrix")
    table, ld, code = _matrix(table, "the table")
    dev = table.device
    ids = _ids(ids, dev)
    V, d = table.shape
    out = _rows_like(ids.shape, d, table)
    here, stream = launch_on(dev)
    with here:
        check(_lib.load().lamq_embedding_lookup(
            table.data_ptr(), code, ld, V, d, ids.data_ptr(), ids.dtype is torch.int64, ids.numel(), scale,
            _padding(padding_idx, V), out.data_ptr(), d, _STATUS.on(dev).data_ptr(), stream), "lamq_embedding_lookup")
    return out


def lookup_gradient(grad: torch.Tensor, ids: torch.Tensor, rows: int, scale: float = 1.0,
                    padding_idx: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of `lookup` in a table of `rows` rows: row v is scale · the sum of `grad` (ids.shape + (d,), fp32
    or bf16) over the tokens with id v, in fp32, rounded once to grad's type. With `out` (rows x d, grad's type) the
    gradient is added to it and rows without a token are left alone. Equal calls give equal bits."""
    if grad.shape[:-1] != ids.shape or grad.ndim < 1:
        raise ValueError(f"one gradient row per id: gradient {tuple(grad.shape)}, ids {tuple(ids.shape)}")
    if rows < 0:
        raise ValueError("rows must not be negative")
    d = grad.shape[-1]
    grad, ld, code = _matrix(grad if grad.ndim == 2 else grad.reshape(ids.numel(), d), "the gradient")
    dev = grad.device
    ids = _ids(ids, dev)
    accumulate = out is not None
    if accumulate:
        if out.shape != (rows, d) or out.dtype != grad.dtype or out.device != dev or out.stride(-1) != 1 or (
                rows > 1 and out.stride(0) < d):
            raise ValueError(f"out must be a {rows} x {d} {grad.dtype} matrix with contiguous rows on {dev}")
    else:
        out = _rows_like((rows,), d, grad)
    lib = _lib.load()
    n = ids.numel()
    size = lib.lamq_embedding_gradient_workspace_size(n, d)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    here, stream = launch_on(dev)
    with here:
        check(lib.lamq_embedding_gradient(
            grad.data_ptr(), code, ld, ids.data_ptr(), ids.dtype is torch.int64, n, rows, d, scale,
            _padding(padding_idx, rows), accumulate, out.data_ptr(), max(out.stride(0), d), ptr(ws), size,
            _STATUS.on(dev).data_ptr(), stream), "lamq_embedding_gradient")
    return out


class _ScaledEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, padding_idx, zeros):
        _padding(padding_idx, table.shape[0])
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale, ctx.padding_idx = table.shape[0], scale, padding_idx
        # without `zeros` the padding token's row as it is stored; its gradient stays zero in both
        return lookup(table, ids, scale, padding_idx if zeros else None)

    @staticmethod
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        return _ScaledGradient.apply(grad, ids, ctx.rows, ctx.scale, ctx.padding_idx), None, None, None, None


class _ScaledGradient(torch.autograd.Function):
    """`lookup_gradient`, linear in its rows: its own gradient is a lookup, with zeros for the tokens that add nothing."""

    @staticmethod
    def forward(ctx, grad, ids, rows, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.scale, ctx.padding_idx = scale, padding_idx
        return lookup_gradient(grad, ids, rows, scale, padding_idx)

    @staticmethod
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        return _ScaledEmbedding.apply(grad, ids, ctx.scale, ctx.padding_idx, True), None, None, None, None


def scaled_embedding(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None):
    """scale · table[ids] under autograd, as torch's embedding: tokens with id `padding_idx` get the stored row (not
    `lookup`'s zeros) and add nothing to the table's gradient, which is `lookup_gradient`."""
    return _ScaledEmbedding.apply(table, ids, float(scale), padding_idx, False)
