"""The step operators' structs and workspaces as the library sees them (no GPU needed)."""

import ctypes
import random

import pytest
from test_step_abi import N, P, lib, norm  # noqa: F401  (lib: the loaded library)

from lookatmyquant_b200 import _lib

_c = ctypes
ROWS = [("data", _c.c_void_p), ("inner", _c.c_int64), ("row", _c.c_int64), ("outer", _c.c_int64)]


class Rows(_c.Structure):
    _fields_ = ROWS


class NormArgs(_c.Structure):
    """The header's declaration, laid out by C's rules (the library asserts the sizes and places of its own)."""
    _fields_ = [("rows", _c.c_int64), ("gate_span", _c.c_int64),
                *((k, _c.c_int) for k in ("d", "residual_dtype", "branch_dtype", "weight_dtype", "post_dtype", "gate_dtype")),
                *((k, _c.c_float) for k in ("scale", "eps", "offset")), ("reserved", _c.c_int), ("residual", Rows), ("branch", Rows),
                *((k, _c.c_void_p) for k in ("weight", "post", "gate", "h", "y")), ("dh", Rows), ("dy", Rows),
                *((k, _c.c_void_p) for k in ("d_residual", "d_branch", "d_weight", "d_post", "d_gate"))]


class Gradient(_c.Structure):
    _fields_ = [("data", _c.c_void_p), ("out", _c.c_void_p), ("n", _c.c_int64), ("dtype", _c.c_int), ("out_dtype", _c.c_int)]


@pytest.mark.parametrize("packed,struct,size", [(_lib.NORM_ARGS, NormArgs, 264), (_lib.GRADIENT, Gradient, 32)])
def test_what_the_bindings_pack_lies_where_the_header_says(packed, struct, size):
    assert packed.size == ctypes.sizeof(struct) == size

    def flat(s):
        for name, kind in s._fields_:
            x = getattr(s, name)
            yield from flat(x) if isinstance(x, ctypes.Structure) else [0 if x is None else x]
    count = len(list(flat(struct())))
    numbers = list(range(1, count + 1))
    assert [int(x) for x in flat(struct.from_buffer_copy(packed.pack(*numbers)))] == numbers


@pytest.mark.parametrize("seed", range(4))
def test_workspaces_have_room_for_every_partial_row(lib, seed):  # noqa: F811
    """What the sizes that the library returns say of its plan: `grid` partial rows for a weight; of a shared gate none where
    ranges hold its rows whole, as many for a gate of all rows, and otherwise one for each range and gate row that may meet,
    ranges + gate rows - 1 of them."""
    rng = random.Random(seed)
    size = lib.lamq_norm_backward_workspace_size
    kinds = set()
    for _ in range(400):
        d = rng.choice([1, 8, 64, 129, 960, 2560, 4097, 8192, 16384])
        span = int(2 ** rng.uniform(0, 13))
        n = span * rng.randint(1, 60)
        t = dict(n=n, d=d, span=span, gate=P, rt=rng.randint(0, 1), residual=(P, 1 << 30, d, 0), branch=(P, 1 << 30, d, 0),
                 dh=(P, 1 << 30, d, 0), dy=(P, 1 << 30, d, 0))
        t.update(bt=t["rt"] or rng.randint(0, 1))
        row = (d + 7) // 8 * 8 * 4
        gates, both = size(norm(**t, dg=P)), size(norm(**t, dg=P, dw=P))
        assert gates % row == 0 and (both - gates) % row == 0
        grid, partial = (both - gates) // row, gates // row
        assert 1 <= grid <= n
        if span == 1:
            assert partial == 0
        elif span == n:
            assert partial in ((grid,) if n > 1 else (0, grid))
        elif partial and partial != grid:
            assert partial >= grid + n // span - 1
        kinds.add("one" if span == n else "inside" if partial == 0 else "block" if partial == grid else "across")
    assert kinds >= {"one", "inside", "across"}
