"""Rows that begin between two 16-byte pieces: what lies before a tensor's first row and behind its last is not used."""

import pytest
import torch
from test_gpu_norms import BF, FP, N, generator, values  # noqa: F401  (N: the module under test)

pytestmark = pytest.mark.gpu


def between(x, shift, beside):
    """x's values `shift` elements into a buffer, 16 elements of `beside` around them."""
    flat = torch.full((x.numel() + 48,), beside, dtype=x.dtype, device="cuda")
    at = flat[16 + shift:16 + shift + x.numel()].view(x.shape)
    at.copy_(x)
    return at


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d", [1, 2, 3, 5, 37, 64, 129, 1337, 4095, 4097])
def test_what_lies_beside_a_tensor(N, d, dtype):  # noqa: F811
    g = generator(d)
    shape = (2, 7, d)
    for shift in (0, 1, 3, 5, 7):
        parts = [values(g, *shape, dtype=dtype) for _ in range(3)] + [values(g, d, dtype=dtype) for _ in range(2)]
        results = []
        for beside in (0.0, float("nan")):
            x, b, gate, w, u = (between(t, shift, beside) for t in parts)
            h, y = N.join_forward(x, b, w, u, gate, 0.5)
            results.append((h, y, *N.join_backward(x, b, h, b, w, u, gate, 0.5), *N.join_backward(x, None, h, b, None, None, gate),
                            N.norm_forward(x, w), *N.norm_backward(b, x, w)))
        for a, c in zip(*results):
            assert a is None and c is None or torch.equal(a, c) and bool(a.isfinite().all())


def test_rows_far_apart(N):  # noqa: F811
    """The last tokens of two long texts: rows 2^29 + 64 elements apart, in place in the norm, through a copy in a join."""
    stride = 2**29 + 64
    base = torch.empty(stride + 64, dtype=BF, device="cuda")
    x = torch.as_strided(base, (2, 64), (stride, 1))
    x.copy_(values(generator(1), 2, 64))
    w = values(generator(2), 64, dtype=BF)
    near = x.contiguous()
    assert torch.equal(N.norm_forward(x, w), N.norm_forward(near, w))
    for a, b in zip((*N.join_forward(x, x, w), *N.join_backward(x, x, x, x, w), *N.norm_backward(x, x, w)),
                    (*N.join_forward(near, near, w), *N.join_backward(near, near, near, near, w), *N.norm_backward(near, near, w))):
        assert a is None and b is None or torch.equal(a, b)
