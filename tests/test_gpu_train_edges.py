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


POLAR = [(8.28721201814563, -23.595886519098837, 17.300387312530933),
         (4.107059111542203, -2.9478499167379106, 0.5448431082926601),
         (3.9486908534822946, -2.908902115962949, 0.5518191394370137),
         (3.3184196573706015, -2.488488024314874, 0.51004894012372),
         (2.300652019954817, -1.6689039845747493, 0.4188073119525673)]


@pytest.mark.parametrize("scale", [1.0, 1.01])
@pytest.mark.parametrize("m,n,rank,noise", [(320, 960, 4, 1.0), (150, 2000, 2, 3.0), (2000, 150, 2, 3.0), (256, 512, 256, 1.0)])
def test_steep_schedules_are_as_exact_as_muons(m, n, rank, noise, scale):
    """A published schedule whose first step multiplies a small rounding by 24, within the tolerance of Muon's coefficients:
    the bf16 output's rounding (at most 2^-8 of each entry, uniform) and ten roundings of 2^-11."""
    from lookatmyquant_b200 import orthogonal as N
    g = torch.Generator("cuda").manual_seed(m + n)
    G = 1e-3 * (torch.randn(m, rank, device="cuda", generator=g) @ torch.randn(rank, n, device="cuda", generator=g)
                + noise * torch.randn(m, n, device="cuda", generator=g))
    abc = [(a / scale, b / scale**3, c / scale**5) for a, b, c in POLAR]
    X = G.double() / (G.double().norm() + 1e-7)
    X = X.T if m > n else X
    for a, b, c in abc:
        A = X @ X.T
        X = a * X + (b * A + c * A @ A) @ X
    X = X.T if m > n else X
    got = N.newton_schulz(G, coefficients=abc)
    assert float((got.double() - X).norm()) <= math.hypot(2.0**-8, 10 * 2.0**-11) / math.sqrt(3) * float(X.norm())
    N.check_status()
