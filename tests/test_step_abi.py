"""The step operators' C ABI (include/lamq_b200_step.h): every declared symbol is exported and bound, and arguments are checked
before the device is touched (no GPU needed)."""

import re
import struct
from pathlib import Path

import pytest

from lookatmyquant_b200 import _lib
from lookatmyquant_b200.build import LIB, build

HEADER = Path(__file__).resolve().parents[1] / "include" / "lamq_b200_step.h"
N, P = None, 4096  # P: a non-null pointer that the checks never dereference


@pytest.fixture(scope="module")
def lib():
    if not LIB.exists():
        build()
    return _lib.load()


def rows(data=P, inner=1 << 30, row=64, outer=0):
    return data, inner, row, outer


def norm(n=6, span=1, d=64, rt=0, bt=0, wt=0, pt=0, gt=0, scale=1.0, eps=1e-6, offset=0.0, residual=rows(), branch=rows(),
         weight=P, post=0, gate=0, h=P, y=P, dh=rows(), dy=rows(), dr=P, db=P, dw=0, du=0, dg=0):
    return _lib.NORM_ARGS.pack(n, span, d, rt, bt, wt, pt, gt, scale, eps, offset, 0, *residual, *branch, weight, post, gate, h,
                               y, *dh, *dy, dr, db, dw, du, dg)


NO = rows(0, 1, 0)
BOTH = [(N, b"null pointer (args)"), (norm(n=-1), b"bad shape"), (norm(d=-1), b"bad shape"), (norm(n=2**31), b"bad shape"),
        (norm(d=16385), b"up to 16384"), (norm(rt=2), b"dtype"), (norm(gt=7), b"dtype"), (norm(rt=1, bt=0), b"dtype"),
        (norm(rt=0, bt=1, branch=NO), b"dtype"), (norm(eps=0.0), b"eps"), (norm(eps=float("nan")), b"eps"),
        (norm(scale=float("inf")), b"finite"), (norm(offset=float("nan")), b"finite"), (norm(gate=P, span=4), b"divide"),
        (norm(gate=P, span=0), b"divide"), (norm(residual=rows(0)), b"null pointer (residual)"),
        (norm(residual=rows(inner=0)), b"inner count"), (norm(branch=rows(inner=2**31)), b"inner count"),
        (norm(branch=rows(inner=2, outer=100)), b"one stride"), (norm(residual=rows(row=2**30)), b"one stride"),
        (norm(branch=NO, weight=0), b"the norm alone"), (norm(branch=NO, post=P), b"the norm alone"),
        (norm(branch=NO, gate=P, span=6), b"the norm alone")]
INVALID = [("lamq_norm_forward", (a, N), text) for a, text in BOTH + [(norm(h=0), b"null pointer (h)"),
                                                                      (norm(y=0), b"null pointer (y)")]]
INVALID += [("lamq_norm_backward", (a, P, 1 << 40, N), text) for a, text in BOTH + [
    (norm(dr=0), b"null pointer (d_residual)"), (norm(branch=NO, db=0), b"no dh"), (norm(branch=NO, dh=NO), b"no d_branch"),
    (norm(branch=NO, dh=NO, dy=NO), b"null pointer (dy)"),
    (norm(weight=0), b"belong to a weight"), (norm(weight=0, dy=NO, dw=P), b"belong to a weight"),
    (norm(du=P), b"belongs to a post weight"), (norm(dg=P), b"belongs to a gate"), (norm(dy=rows(inner=-1)), b"inner count")]]
INVALID += [("lamq_norm_backward", (norm(dw=P), P, 0, N), b"workspace of"),
            ("lamq_norm_backward", (norm(dw=P), N, 1 << 40, N), b"null pointer (workspace)"),
            ("lamq_norm_backward", (norm(dw=P), P + 16, 1 << 40, N), b"32-byte aligned")]


def tensors(*entries):
    return struct.pack("=" + "2Qq2i" * len(entries), *(x for e in entries for x in e))


ONE = tensors((P, P, 10, 0, 0))
LISTS = [(N, 2, b"null pointer (list)"), (ONE, -1, b"bad shape"), (tensors((P, P, -1, 0, 0)), 1, b"bad shape"),
         (tensors((P, P, 2**43 + 1, 0, 0)), 1, b"bad shape"), (tensors((P, P, 2**42, 0, 0)) * 3, 3, b"more than 2^43"),
         (tensors((P, P, 4, 2, 0)), 1, b"dtype"), (tensors((0, P, 4, 0, 0)), 1, b"null pointer (tensor 0)")]
INVALID += [("lamq_gradient_norm", (a, n, P, P, 1 << 40, N), text) for a, n, text in LISTS]
INVALID += [("lamq_gradient_clip", (a, n, 1.0, 1e-6, P, P, 1 << 40, N), text) for a, n, text in LISTS + [
    (tensors((P, P, 4, 0, 1)), 1, b"in place"), (tensors((P, P, 4, 0, 5)), 1, b"dtype"),
    (tensors((P, 0, 4, 0, 0)), 1, b"null pointer (tensor 0)"),
    (ONE * 2, 2, b"overlap"),                                                         # the same tensor twice
    (tensors((P, P, 10, 0, 0), (P + 36, P + 36, 10, 0, 0)), 2, b"overlap"),           # its end
    (tensors((P, 2 * P, 10, 0, 0), (2 * P + 4, 4 * P, 10, 0, 0)), 2, b"overlap"),     # an output over another's input
    (tensors((P, 2 * P, 10, 0, 0), (4 * P, 2 * P + 16, 10, 1, 1)), 2, b"overlap"),    # two outputs
    (tensors((P, P + 4, 10, 0, 0)), 1, b"overlap")]]                                  # an output beside its own input
INVALID += [("lamq_gradient_norm", (ONE, 1, N, P, 1 << 40, N), b"null pointer (norm)"),
            ("lamq_gradient_norm", (ONE, 1, P, P, 16, N), b"workspace of"),
            ("lamq_gradient_norm", (ONE, 1, P, N, 1 << 40, N), b"null pointer (workspace)"),
            ("lamq_gradient_clip", (ONE, 1, -1.0, 1e-6, P, P, 1 << 40, N), b"max_norm"),
            ("lamq_gradient_clip", (ONE, 1, float("nan"), 1e-6, P, P, 1 << 40, N), b"max_norm"),
            ("lamq_gradient_clip", (ONE, 1, 1.0, -1.0, P, P, 1 << 40, N), b"eps"),
            ("lamq_gradient_clip", (ONE, 1, 1.0, 1e-6, P, P, 16, N), b"workspace of")]

EMPTY = [("lamq_norm_forward", (norm(n=0, residual=NO, h=0, y=0), N)), ("lamq_norm_forward", (norm(d=0, residual=NO), N)),
         ("lamq_norm_backward", (norm(n=0, residual=NO, dr=0), N, 0, N)),
         ("lamq_norm_backward", (norm(d=0, dw=P, residual=NO), N, 0, N))]


def test_every_declared_symbol_is_exported(lib):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    declared = set(re.findall(r"\b(lamq_[a-z0-9_]+)\s*\(", text))
    for name in declared:
        assert hasattr(lib, name) and name in _lib.SIGNATURES, name
    assert {n for n in declared if not n.endswith("_workspace_size")} == {c[0] for c in INVALID}


@pytest.mark.parametrize("name,args,text", INVALID, ids=[f"{c[0]}-{i}" for i, c in enumerate(INVALID)])
def test_entry_point_rejects_bad_arguments(lib, name, args, text):
    before = lib.lamq_kernel_launches()
    assert getattr(lib, name)(*args) == _lib.LAMQ_ERR_INVALID
    assert text in lib.lamq_last_error(), lib.lamq_last_error()
    assert lib.lamq_kernel_launches() == before


@pytest.mark.parametrize("name,args", EMPTY, ids=[f"{c[0]}-{i}" for i, c in enumerate(EMPTY)])
def test_entry_point_accepts_empty_input(lib, name, args):
    before = lib.lamq_kernel_launches()
    assert getattr(lib, name)(*args) == _lib.LAMQ_OK
    assert lib.lamq_kernel_launches() == before


def test_norm_args_layout_matches_the_header():
    assert _lib.NORM_ARGS.size == 264 and "264 bytes" in HEADER.read_text()


def test_workspaces(lib):
    size = lib.lamq_norm_backward_workspace_size
    assert size(norm()) == 0 == size(norm(n=0, dw=P)) == size(norm(d=16385, dw=P))
    one = size(norm(n=10_000, dw=P))
    assert one > 0 and one % (64 * 4) == 0
    # a gate for each row is written at once, one for all is summed like a weight, one for 5000 rows leaves partials
    assert size(norm(n=10_000, gate=P, dg=P, span=1)) == 0
    assert size(norm(n=10_000, gate=P, dg=P, span=10_000)) > 0 and size(norm(n=10_000, gate=P, dg=P, span=5_000)) > 0
    assert lib.lamq_gradient_workspace_size(0) == 0 < lib.lamq_gradient_workspace_size(1)
    assert lib.lamq_gradient_workspace_size(1001) == 2 * lib.lamq_gradient_workspace_size(1000)


@pytest.mark.parametrize("seed", range(4))
def test_gate_partials_stay_inside_the_workspace(seed):
    """A worker (a range of rows) and a gate row meet in the partial row worker + gate row: no two pairs in one, none behind
    workers + gate rows, and a gate row's partials are one run. (The indices of the kernel and of its sums, for many plans.)"""
    import random
    rng = random.Random(seed)
    for _ in range(300):
        per, span = rng.randint(1, 40), rng.randint(1, 90)
        n = span * rng.randint(1, 30)
        seen = {}
        for row in range(n):
            seen.setdefault((row // per, row // span), len(seen))
        workers, gates = -(-n // per), n // span
        slots = [k + g for k, g in seen]
        assert len(set(slots)) == len(slots) and max(slots) < workers + gates
        for g in range(gates):
            k0, k1 = g * span // per, (g * span + span - 1) // per
            assert [k + g for k, q in seen if q == g] == list(range(k0 + g, k1 + g + 1))
