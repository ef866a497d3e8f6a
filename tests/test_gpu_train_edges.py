"""The training operators at the edges of what their callers may pass."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_attention_takes_contiguous_tensors_that_start_anywhere():
    """A contiguous view that begins between two 16-byte pieces (a slice of a flat buffer) is copied like any other that TMA
    cannot read in place."""
    from lookatmyquant_b200 import attention as A
    g = torch.Generator("cuda").manual_seed(1)
    q, k, v, do = (torch.randn(2, H, 150, 64, device="cuda", generator=g).bfloat16() for H in (4, 2, 2, 4))
    o, lse = A.forward(q, k, v)
    want = (o, lse, *A.backward(do, q, k, v, o, lse))

    def moved(x):
        flat = torch.zeros(x.numel() + 3, dtype=x.dtype, device=x.device)
        y = flat[3:].view(x.shape)
        y.copy_(x)
        assert y.is_contiguous() and y.data_ptr() % 16
        return y
    q, k, v, do = map(moved, (q, k, v, do))
    o, lse = A.forward(q, k, v)
    for a, b in zip((o, lse, *A.backward(do, q, k, v, moved(o.contiguous()), lse)), want):
        assert torch.equal(a, b)
