"""Pointers that do not lie at a multiple of their element's size (a double's for the gradients' workspace) are refused before the
device is touched, where they would end the context with a misaligned address (no GPU needed)."""

import pytest
from test_step_abi import N, NO, P, lib, norm, rows, tensors  # noqa: F401  (lib: the loaded library)

from lookatmyquant_b200 import _lib

BIG = 1 << 40
FORWARD = [("residual", norm(residual=rows(P + 2))), ("branch", norm(branch=rows(P + 1), bt=1)), ("weight", norm(weight=P + 2)),
           ("post", norm(post=P + 1, pt=1)), ("gate", norm(gate=P + 3, gt=1)), ("gate", norm(gate=P + 2, gt=0)),
           ("h", norm(h=P + 2)), ("y", norm(y=P + 1, bt=1)), ("residual", norm(residual=rows(P + 1), rt=1, bt=1, branch=NO))]
BACKWARD = [("residual", norm(residual=rows(P + 2))), ("dh", norm(dh=rows(P + 2))), ("dy", norm(dy=rows(P + 1), bt=1)),
            ("d_residual", norm(dr=P + 2)), ("d_branch", norm(db=P + 1, bt=1)), ("d_weight", norm(dw=P + 2)),
            ("d_post", norm(post=P, du=P + 1, pt=1)), ("d_gate", norm(gate=P, dg=P + 2))]
CALLS = [("lamq_norm_forward", (a, N), f"{w}: not aligned") for w, a in FORWARD]
CALLS += [("lamq_norm_backward", (a, P, BIG, N), f"{w}: not aligned") for w, a in BACKWARD]
ONE = tensors((P, P, 10, 0, 0))
for name, args in (("lamq_gradient_norm", ()), ("lamq_gradient_clip", (1.0, 1e-6))):
    CALLS += [(name, (ONE, 1, *args, P, P + 4, BIG, N), "8-byte aligned"), (name, (ONE, 1, *args, P + 2, P, BIG, N), "norm: not aligned")]
    for data, out, types in ((P + 2, P + 2, (0, 0)), (P + 1, P + 1, (1, 1))):
        bad = tensors((P, P, 3, 0, 0), (data + 64, out + 64, 10, *types))
        CALLS.append((name, (bad, 2, *args, P, P, BIG, N), "tensor 1: not aligned"))
CALLS += [("lamq_gradient_clip", (tensors((P, 2 * P + o, 10, 0, t)), 1, 1.0, 1e-6, P, P, BIG, N), "tensor 0: not aligned")
          for o, t in ((2, 0), (1, 1))]


@pytest.mark.parametrize("name,args,text", CALLS, ids=[f"{c[0]}-{i}" for i, c in enumerate(CALLS)])
def test_misaligned_pointers_are_refused(lib, name, args, text):  # noqa: F811
    before = lib.lamq_kernel_launches()
    assert getattr(lib, name)(*args) == _lib.LAMQ_ERR_INVALID
    assert text.encode() in lib.lamq_last_error(), lib.lamq_last_error()
    assert lib.lamq_kernel_launches() == before
