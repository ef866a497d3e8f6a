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


def test_keys_without_query_heads_get_zero_gradients():
    from lookatmyquant_b200 import attention as A
    q, k = torch.zeros(1, 0, 5, 64, device="cuda").bfloat16(), torch.randn(1, 2, 9, 64, device="cuda").bfloat16()
    for _ in range(3):
        torch.full((1 << 16,), math.nan, device="cuda")  # what the allocator hands out next holds no zeros
        dq, dk, dv = A.backward(q, q, k, k, *A.forward(q, k, k))
        assert dq.shape == q.shape and dk.shape == dv.shape == k.shape
        assert float(dk.abs().sum()) == float(dv.abs().sum()) == 0


def test_empty_shapes_of_any_rank():
    """Shapes with an axis of none come back as they are: no axis's length is to be guessed from no elements."""
    from lookatmyquant_b200 import embedding as E, orthogonal as N
    for shape in ((2, 3, 0, 4), (2, 3, 4, 0), (2, 0, 3, 4), (0, 2, 0, 0)):
        assert N.newton_schulz(torch.zeros(shape, device="cuda")).shape == shape
    ids = torch.zeros(2, 3, dtype=torch.long, device="cuda")
    assert E.lookup(torch.zeros(5, 0, device="cuda"), ids).shape == (2, 3, 0)
    assert E.lookup_gradient(torch.zeros(2, 3, 0, device="cuda"), ids, 5).shape == (5, 0)
    assert E.lookup_gradient(torch.zeros(2, 0, 4, device="cuda"), ids[:, :0], 5).shape == (5, 4)


def test_newton_schulz_of_matrices_at_the_end_of_fp32():
    """Without an eps: a zero matrix gives zeros, and a matrix is its own multiple's (a power of two takes no bits) down to
    where fp32 ends. Norms of about 7e-2 · 2^-k."""
    from lookatmyquant_b200 import orthogonal as N
    G = (torch.randn(60, 90, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) * 1e-3)
    G = G.bfloat16().float()  # 8 bits, so that they survive as subnormals
    G = torch.where(G.abs() < 2.0**-16, 0.0, G)
    want = N.newton_schulz(G, eps=0.0)
    for k in (60, 100, 115, 125):
        assert torch.equal(N.newton_schulz(G * 2.0**-k, eps=0.0), want), k
    assert float(N.newton_schulz(torch.zeros(40, 60, device="cuda"), eps=0.0).abs().sum()) == 0
    N.check_status()
