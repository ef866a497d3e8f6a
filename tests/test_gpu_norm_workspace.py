"""What a backward call writes and reads of its workspace: every byte behind it stays, and nothing is read that was not written."""

import random

import pytest
import torch
from step_reference import assert_close, join_backward
from test_gpu_norms import BF, FP, generator, values

pytestmark = pytest.mark.gpu

GUARD = 1 << 20


@pytest.mark.parametrize("seed", range(6))
def test_partial_rows_stay_inside_the_workspace(seed):
    """Plans of random rows, spans, widths and types, all parameters' gradients wanted; the workspace's size to the byte, NaN
    inside, a pattern behind."""
    from lookatmyquant_b200 import _lib
    lib, rng = _lib.load(), random.Random(seed)
    for _ in range(25):
        d = rng.choice([1, 8, 24, 64, 129, 256, 960, 2560, 4097, 5120, 8200])
        span = int(2 ** rng.uniform(0, 10))
        n = span * rng.randint(1, max(1, min(40, 6000 // span)))
        r, b = rng.choice([(BF, BF), (FP, BF), (FP, FP)])
        g = generator(rng.randrange(1 << 30))
        texts = n // span
        h, branch, dh, dy = (values(g, texts, span, d, dtype=t) for t in (r, b, r, b))
        w, u = values(g, d), values(g, d, dtype=BF)
        gate = values(g, texts, 1, d, dtype=b)
        outs = [torch.empty_like(x) for x in (h, branch, w, u, gate)]
        rows = lambda x: (x.data_ptr(), 1 << 30, d, 0)
        code = {FP: 0, BF: 1}
        args = _lib.NORM_ARGS.pack(n, span, d, code[r], code[b], 0, 1, code[b], 0.5, 1e-5, 0.0, 0, *rows(h), *rows(branch),
                                   w.data_ptr(), u.data_ptr(), gate.data_ptr(), 0, 0, *rows(dh), *rows(dy),
                                   *(x.data_ptr() for x in outs))
        size = lib.lamq_norm_backward_workspace_size(args)
        ws = torch.full(((size + GUARD) // 4,), float("nan"), device="cuda")
        ws[size // 4:] = 7.0
        _lib.check(lib.lamq_norm_backward(args, ws.data_ptr(), size, _lib.stream_ptr()), "lamq_norm_backward")
        assert bool((ws[size // 4:] == 7.0).all())
        want = join_backward(dh, dy, h, branch, w, u, gate, 0.5, 1e-5)
        for got, name in zip(outs, ("residual", "branch", "weight", "post", "gate")):
            assert_close(got, want[name], f"d_{name} of {texts} x {span} x {d}")


@pytest.mark.parametrize("n,d", [(840_000, 2560), (132_000, 16384)])
@pytest.mark.parametrize("gate", ["text", "token"])
def test_joins_of_many_rows(n, d, gate):
    """Offsets behind 2^31 elements in every tensor of a join and its gradients: zeros, but for the last rows."""
    from lookatmyquant_b200 import norms as N
    from step_reference import join_forward
    last = 3

    def rows(seed, scale=1.0):
        x = torch.zeros(2, n // 2, d, dtype=BF, device="cuda")
        x[-1, -last:] = values(generator(seed), last, d, scale=scale, dtype=BF)
        return x
    stream, branch = rows(1), rows(2)
    w, u = values(generator(3), d, dtype=BF), values(generator(4), d, dtype=BF)
    gates = rows(5) if gate == "token" else values(generator(5), 2, 1, d, dtype=BF)
    end = lambda x: x[-1:, -last:]
    ends = (end(stream), end(branch), w, u, end(gates) if gate == "token" else gates[-1:])
    h, y = N.join_forward(stream, branch, w, u, gates, 0.5)
    wh, wy = join_forward(*ends, 0.5)
    assert_close(end(h), wh, "h")
    assert_close(end(y), wy, "y")
    assert not bool(h[0].any()) and not bool(y[0].any()) and not bool(y[1, :100].any())
    del y
    dh, dy = rows(6, 1e-3), rows(7, 1e-3)
    got = dict(zip(("residual", "branch", "weight", "post", "gate"), N.join_backward(dh, dy, h, branch, w, u, gates, 0.5)))
    want = join_backward(end(dh), end(dy), end(h), *ends[1:], 0.5)
    for k in ("weight", "post"):
        assert_close(got[k], want[k], f"d_{k}")
    for k in ("residual", "branch"):
        assert_close(end(got[k]), want[k], f"d_{k}")
        assert not bool(got[k][0].any()) and not bool(got[k][1, :-last].any())
    d_gate = got["gate"]
    assert_close(end(d_gate) if gate == "token" else d_gate[-1:], want["gate"], "d_gate")
    assert not bool(d_gate[0].any())
