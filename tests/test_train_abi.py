"""The training operators' C ABI (include/lamq_b200_train.h): every declared symbol is exported and bound, arguments
are checked before the device is touched, and empty inputs are a successful no-op (no GPU needed)."""

import ctypes
import re
import struct
from pathlib import Path

import pytest

from lookatmyquant_b200 import _lib
from lookatmyquant_b200.build import LIB, build

HEADER = Path(__file__).resolve().parents[1] / "include" / "lamq_b200_train.h"
N, P = None, 4096  # P: a non-null pointer that the checks never dereference


def declared():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return sorted(set(re.findall(r"\b(lamq_[a-z0-9_]+)\s*\(", text)))


@pytest.fixture(scope="module")
def lib():
    if not LIB.exists():
        build()
    return _lib.load()


INVALID = [
    ("lamq_embedding_lookup", (P, 0, 4, 10, 8, P, 1, 5, 1.0, -1, P, 8, P, N), b"bad shape"),
    ("lamq_embedding_lookup", (P, 2, 8, 10, 8, P, 1, 5, 1.0, -1, P, 8, P, N), b"dtype"),
    ("lamq_embedding_lookup", (P, 0, 8, 10, 8, N, 1, 5, 1.0, -1, P, 8, P, N), b"null pointer"),
    ("lamq_embedding_lookup", (P, 0, 8, 10, 8, P, 1, 5, 1.0, -1, P, 8, N, N), b"null pointer"),
    ("lamq_embedding_lookup", (P, 0, 8, 10, 8, P, 1, 2**40, 1.0, -1, P, 8, P, N), b"too many tokens"),
    ("lamq_embedding_gradient", (P, 0, 8, P, 1, -1, 10, 8, 1.0, -1, 0, P, 8, P, 0, P, N), b"bad shape"),
    ("lamq_embedding_gradient", (P, 7, 8, P, 1, 4, 10, 8, 1.0, -1, 0, P, 8, P, 0, P, N), b"dtype"),
    ("lamq_embedding_gradient", (P, 0, 8, P, 1, 2**33, 10, 8, 1.0, -1, 0, P, 8, P, 0, P, N), b"more than 2^31"),
    ("lamq_embedding_gradient", (N, 0, 8, P, 1, 4, 10, 8, 1.0, -1, 0, P, 8, P, 0, P, N), b"null pointer"),
    ("lamq_embedding_gradient", (P, 0, 8, P, 1, 2049, 10, 8, 1.0, -1, 0, P, 8, P, 16, P, N), b"workspace"),
]



def heads(data=P, batch=4096, head=128, row=512):
    return (data, batch, head, row)


def attention(batch=2, heads_=4, kv=2, D=64, Lq=9, Lk=9, scale=0.125, q=heads(), k=heads(), v=heads(), o=heads(), lse=P,
              d_o=heads(), dq=heads(), dk=heads(), dv=heads()):
    return _lib.ATTENTION_ARGS.pack(batch, heads_, kv, D, 1, Lq, Lk, scale, 0, 0, 0, *q, *k, *v, *o, lse, *d_o, *dq, *dk,
                                    *dv)


INVALID += [(f"lamq_attention_{way}", (a, *rest), text)
            for way, rest in (("forward", (P, N)), ("backward", (P, 0, P, N)))
            for a, text in [(N, b"null pointer"), (attention(Lq=-1), b"bad shape"), (attention(D=12), b"head_dim"),
                            (attention(D=136), b"head_dim"), (attention(kv=3), b"not a multiple of 3"),
                            (attention(scale=0.0), b"scale"), (attention(scale=float("nan")), b"scale"),
                            (attention(Lk=2**31), b"lengths up to"), (attention(batch=2**20), b"heads in all"),
                            (attention(q=heads(0)), b"null pointer (q)"), (attention(k=heads(P + 8)), b"aligned"),
                            (attention(v=heads(row=60)), b"multiples of 8"), (attention(o=heads(head=0)), b"positive"),
                            (attention(lse=0), b"null pointer (lse)")]]
INVALID += [("lamq_attention_forward", (attention(), N, N), b"null pointer (status)"),
            ("lamq_attention_backward", (attention(), P, 0, N, N), b"null pointer (status)"),
            ("lamq_attention_backward", (attention(d_o=heads(0)), P, 0, P, N), b"null pointer (do)"),
            ("lamq_attention_backward", (attention(dv=heads(row=-8)), P, 0, P, N), b"positive"),
            ("lamq_attention_backward", (attention(), P, 100, P, N), b"workspace of 8192 bytes")]

C3 = struct.pack("3f", 3.4445, -4.7750, 2.0315)
INVALID += [("lamq_newton_schulz", (P, dt, ld, 64, b, m, n, steps, coef, eps, out, ws, 0, P, N), text)
            for dt, ld, b, m, n, steps, coef, eps, out, ws, text in [
                (0, 8, 1, -1, 8, 1, C3, 0.0, P, P, b"bad shape"), (0, 7, 1, 8, 8, 1, C3, 0.0, P, P, b"bad shape"),
                (2, 8, 1, 8, 8, 1, C3, 0.0, P, P, b"dtype"), (0, 8, 1, 8, 8, 0, C3, 0.0, P, P, b"1 to 16 steps"),
                (0, 8, 1, 8, 8, 17, C3, 0.0, P, P, b"1 to 16 steps"), (0, 8, 1, 8, 8, 1, C3, -1.0, P, P, b"eps"),
                (0, 8, 2, 9, 8, 1, C3, 0.0, P, P, b"overlap"), (0, 8, 1, 8, 8, 1, N, 0.0, P, P, b"null pointer"),
                (0, 2**24, 65535, 2**24, 2**24, 1, C3, 0.0, P, P, b"too large"),
                (0, 8, 1, 8, 8, 1, C3, 0.0, N, P, b"null pointer"), (0, 8, 1, 8, 8, 1, C3, 0.0, P, P, b"workspace")]]

EMPTY = [
    ("lamq_newton_schulz", (N, 0, 8, 0, 0, 8, 8, 1, N, 0.0, N, N, 0, N, N)),
    ("lamq_newton_schulz", (N, 0, 8, 0, 1, 0, 8, 1, N, 0.0, N, N, 0, N, N)),
    ("lamq_attention_forward", (attention(batch=0), N, N)),
    ("lamq_attention_forward", (attention(Lq=0, q=heads(0), o=heads(0)), P, N)),
    ("lamq_attention_backward", (attention(heads_=0), N, 0, N, N)),
    ("lamq_attention_backward", (attention(Lq=0, Lk=0), N, 0, P, N)),
    ("lamq_embedding_lookup", (N, 0, 8, 10, 8, N, 1, 0, 1.0, -1, N, 8, N, N)),
    ("lamq_embedding_gradient", (N, 0, 8, N, 1, 4, 0, 8, 1.0, -1, 0, N, 8, N, 0, N, N)),
]


def test_every_declared_symbol_is_exported(lib):
    for name in declared():
        assert hasattr(lib, name) and name in _lib.SIGNATURES, name


@pytest.mark.parametrize("name,args,text", INVALID, ids=[f"{c[0]}-{i}" for i, c in enumerate(INVALID)])
def test_entry_point_rejects_bad_arguments(lib, name, args, text):
    before = lib.lamq_kernel_launches()
    assert getattr(lib, name)(*args) == _lib.LAMQ_ERR_INVALID
    assert text in lib.lamq_last_error()
    assert lib.lamq_kernel_launches() == before


@pytest.mark.parametrize("name,args", EMPTY, ids=[f"{c[0]}-{i}" for i, c in enumerate(EMPTY)])
def test_entry_point_accepts_empty_input(lib, name, args):
    before = lib.lamq_kernel_launches()
    assert getattr(lib, name)(*args) == _lib.LAMQ_OK
    assert lib.lamq_kernel_launches() == before


def test_tables_cover_every_compute_entry_point():
    compute = {n for n in declared() if not n.endswith("_workspace_size")}
    assert compute <= {c[0] for c in INVALID} & {c[0] for c in EMPTY}


def test_gradient_workspace_size(lib):
    size = lib.lamq_embedding_gradient_workspace_size
    assert size(0, 64) == size(2048, 64) == 0  # few tokens need none
    assert size(4096, 64) >= 4 * 4 * 4096 + 2 * (4096 // 8) * 64 * 4  # keys and positions twice, a partial per chunk twice


def test_newton_schulz_coefficients_that_leave_the_range(lib):
    """Checked after the workspace (whose size is right here) and before the device: sizes and pointers stand in."""
    need = lib.lamq_newton_schulz_workspace_size(1, 8, 8)
    for c in ((40.0, 0.0, 0.0), (6.0, 0.0, 0.0), (0.0, 0.0, 33.0), (float("nan"), 0.0, 0.0)):
        st = lib.lamq_newton_schulz(P, 0, 8, 64, 1, 8, 8, 1, struct.pack("3f", *c), 0.0, P, P, need, P, None)
        assert st == _lib.LAMQ_ERR_INVALID and b"leave the range" in lib.lamq_last_error(), c


def test_attention_args_layout_matches_the_header(lib):
    """The packed lamq_attention_args reaches the library field for field: the checks name the tensor that breaks."""
    assert _lib.ATTENTION_ARGS.size == 328
    for name in ("q", "k", "v", "o"):
        args = attention(**{name: heads(0)})
        assert lib.lamq_attention_forward(args, P, None) == _lib.LAMQ_ERR_INVALID
        assert f"({name})".encode() in lib.lamq_last_error()
    for name, key in (("do", "d_o"), ("dq", "dq"), ("dk", "dk"), ("dv", "dv")):
        args = attention(**{key: heads(0)})
        assert lib.lamq_attention_backward(args, P, 0, P, None) == _lib.LAMQ_ERR_INVALID
        assert f"({name})".encode() in lib.lamq_last_error()
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_exponential_polynomial_error():
    """The polynomial of the attention's exponentials in fp32 instructions, evaluated as the kernel does (fused multiply-adds
    in fp32): within 3e-7 of 2^x (its six-point Chebyshev interpolation is 1.02e-7 off, each of five roundings up to 6e-8 of a
    partial sum that the next factor, at most 1/2, shrinks)."""
    import numpy as np

    src = (HEADER.parents[1] / "lookatmyquant_b200" / "csrc" / "attention.cu").read_text()
    body = src[src.index("float2 ex2_pair(") :]
    body = body[: body.index("\n}\n")]
    coefficients = [np.float32(m) for m in re.findall(r"make_float2\((0\.\d+|1\.0+\d+)f, \1f\)", body)]
    assert len(coefficients) == 6
    x = np.concatenate([np.linspace(-126, 1, 400_001), np.arange(-126, 2) + 0.5, np.arange(-126, 2)]).astype(np.float32)
    n = (x + np.float32(12582912.0)) - np.float32(12582912.0)
    f = (x - n).astype(np.float64)
    assert np.abs(f).max() <= 0.5
    y = np.full(f.shape, coefficients[0], np.float32)
    for c in coefficients[1:]:
        y = (y.astype(np.float64) * f + np.float64(c)).astype(np.float32)
    got = y.astype(np.float64) * 2.0 ** n.astype(np.float64)
    assert np.abs(got / 2.0 ** x.astype(np.float64) - 1).max() < 3e-7
