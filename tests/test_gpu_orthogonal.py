"""Newton-Schulz orthogonalisation and the Muon step against the iteration in 64 bits.

Tolerance, relative Frobenius norm, from the arithmetic: the bf16 output's rounding is at most uniform over ±2^-8 of
each entry (rms 2^-8/sqrt 3). Products take fp16 operands (rms 2^-11/sqrt 3): X's rounding enters through A by at most
2|b + 2c| = 1.4 and through (bA + cA²)X by 3.5, that matrix's own by 3.5: 5.1 a step, in quadrature, and a direction
may have reached its singular value of 1 after the first step, so four steps' count: 10 in all. X itself, A and A² are
held and multiplied to some 2^-21. With fewer than 16 singular values the roundings need not average out: the worst
case, sqrt 3 times that."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
ABC = (3.4445, -4.7750, 2.0315)
TOL = math.hypot(2.0**-8, 10 * 2.0**-11) / math.sqrt(3)


def exact(G, steps=5, coefficients=None, eps=1e-7):
    X = G.double()
    X = X / (torch.linalg.matrix_norm(X, keepdim=True) + eps)
    for a, b, c in coefficients or [ABC] * steps:
        if X.shape[-2] > X.shape[-1]:
            A = X.mT @ X
            X = a * X + X @ (b * A + c * A @ A)
        else:
            A = X @ X.mT
            X = a * X + (b * A + c * A @ A) @ X
    return X


def check(got, want):
    assert got.shape == want.shape and got.dtype == torch.bfloat16
    few = min(want.shape[-2:]) < 16
    err = torch.linalg.matrix_norm(got.double() - want)
    assert bool((err <= TOL * (math.sqrt(3) if few else 1) * torch.linalg.matrix_norm(want)).all()), \
        float((err / torch.linalg.matrix_norm(want)).max())


def update(*shape, seed=0, rank=4, noise=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    m, n = shape[-2:]
    r = min(rank, m, n)
    G = torch.randn(*shape[:-2], m, r, device="cuda", generator=g) @ torch.randn(*shape[:-2], r, n, device="cuda",
                                                                                generator=g)
    return 1e-3 * (G + noise * torch.randn(*shape, device="cuda", generator=g))


SHAPES = [(1, 1), (1, 7), (7, 1), (5, 3), (16, 16), (64, 200), (200, 64), (127, 129), (129, 257), (257, 129), (300, 300),
          (320, 960), (960, 320), (1, 3000), (511, 1025), (1025, 770), (640, 2049)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", SHAPES)
def test_matches_the_iteration(m, n, dtype):
    from lookatmyquant_b200 import orthogonal as N
    G = update(m, n, seed=m * 5000 + n).to(dtype)
    O = N.newton_schulz(G)
    check(O, exact(G))
    assert torch.equal(O, N.newton_schulz(G))
    N.check_status()


@pytest.mark.parametrize("b,m,n", [(2, 5, 9), (3, 130, 300), (7, 200, 70), (2, 257, 520), (1, 40, 40), (300, 20, 24)])
def test_batches(b, m, n):
    from lookatmyquant_b200 import orthogonal as N
    G = update(b, m, n, seed=b) * torch.logspace(-3, 3, b, device="cuda")[:, None, None]
    O = N.newton_schulz(G)
    check(O, exact(G))
    for i in (0, b - 1):  # a matrix of a batch and alone: the sum of squares is split differently, nothing else
        one = N.newton_schulz(G[i])
        assert float((one.double() - O[i].double()).norm()) <= 2.0**-8 * float(O[i].double().norm())
    assert torch.equal(N.newton_schulz(G.reshape(b, 1, m, n)).reshape(b, m, n), O)
    N.check_status()


@pytest.mark.parametrize("steps", [1, 2, 3, 6, 10])
def test_steps_and_coefficients(steps):
    from lookatmyquant_b200 import orthogonal as N
    G = update(150, 260, seed=steps)
    check(N.newton_schulz(G, steps=steps), exact(G, steps))
    each = [(3.4445 - 0.1 * k, -4.7750 + 0.1 * k, 2.0315 - 0.05 * k) for k in range(steps)]
    check(N.newton_schulz(G, steps=steps, coefficients=each), exact(G, coefficients=each))
    check(N.newton_schulz(G, steps=steps, coefficients=[1.5, -0.5, 0.0]), exact(G, coefficients=[(1.5, -0.5, 0.0)] * steps))


@pytest.mark.parametrize("rank,noise", [(1, 0.0), (20, 0.0), (20, 1e-4), (3, 1e-2)])
def test_low_rank_updates(rank, noise):
    """Directions that hold nothing must not fill with the rounding of those that do."""
    from lookatmyquant_b200 import orthogonal as N
    G = update(400, 700, seed=rank, rank=rank, noise=noise)
    got, want = N.newton_schulz(G), exact(G)
    err = float((got.double() - want).norm() / want.norm())
    assert err <= TOL * (math.sqrt(3) if rank < 16 else 1), err


def test_singular_values_come_near_one():
    from lookatmyquant_b200 import orthogonal as N
    G = update(256, 512, seed=3)
    s = torch.linalg.svdvals(N.newton_schulz(G).double())
    p = torch.linalg.svdvals(G.double()) / float(G.double().norm())
    for _ in range(5):
        p = ABC[0] * p + ABC[1] * p**3 + ABC[2] * p**5
    assert float((s.sort().values - p.sort().values).abs().max()) <= 256**0.5 * TOL  # Weyl: the error's norm at most
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3


def test_memory_orders_and_streams():
    from lookatmyquant_b200 import orthogonal as N
    for dtype in (torch.float32, torch.bfloat16):
        big = update(3, 150, 301, seed=1).to(dtype)
        want = N.newton_schulz(big[1, :130, :200].contiguous())
        for view in (big[1, :130, :200], torch.cat([big[1], big[1]], 1)[:130, :200]):
            assert torch.equal(N.newton_schulz(view), want)
        odd = big[1].flatten()[1:1 + 130 * 301].reshape(130, 301)[:, :200]
        assert torch.equal(N.newton_schulz(odd), N.newton_schulz(odd.contiguous()))
        assert torch.equal(N.newton_schulz(big[1, :130, :200].t()), N.newton_schulz(big[1, :130, :200].t().contiguous()))
        pair = big[::2, :130, :200]
        assert torch.equal(N.newton_schulz(pair), N.newton_schulz(pair.contiguous()))
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got = N.newton_schulz(big[1, :130, :200])
        s.synchronize()
        assert torch.equal(got, want)


def test_two_streams_at_once():
    """Two cooperative launches in flight share the device without sharing a workspace."""
    from lookatmyquant_b200 import orthogonal as N
    a, b = update(300, 900, seed=1), update(500, 400, seed=2)
    want = N.newton_schulz(a), N.newton_schulz(b)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s):
            x = N.newton_schulz(a)
        with torch.cuda.stream(t):
            y = N.newton_schulz(b)
        torch.cuda.synchronize()
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])
    N.check_status()


def test_extremes():
    from lookatmyquant_b200 import orthogonal as N
    assert float(N.newton_schulz(torch.zeros(40, 60, device="cuda")).abs().sum()) == 0
    G = update(60, 90, seed=4)
    for f in (1e-25, 1e30):
        check(N.newton_schulz(G * f, eps=0.0), exact(G * f, eps=0.0))
    check(N.newton_schulz(G * 1e-8), exact(G * 1e-8))  # a norm of the order of eps
    for bad in (math.nan, math.inf):
        x = torch.stack([G, G, G])
        x[1, 3, 4] = bad
        O = N.newton_schulz(x)
        assert bool(O[1].isnan().all()) and torch.equal(O[0], O[2]) and bool(O[0].isfinite().all())
    for shape in ((0, 5), (5, 0), (0, 4, 4), (3, 0, 4)):
        assert N.newton_schulz(torch.zeros(shape, device="cuda")).shape == shape
    N.check_status()


def test_refusals():
    from lookatmyquant_b200 import orthogonal as N
    G = torch.zeros(8, 8, device="cuda")
    for call, err in [(lambda: N.newton_schulz(G.half()), TypeError), (lambda: N.newton_schulz(G.cpu()), TypeError),
                      (lambda: N.newton_schulz(G[0]), ValueError), (lambda: N.newton_schulz(G, steps=0), ValueError),
                      (lambda: N.newton_schulz(G, steps=17), ValueError),
                      (lambda: N.newton_schulz(G, coefficients=[(1.0, 0.0, 0.0)] * 4), ValueError),
                      (lambda: N.newton_schulz(G, coefficients=(1.0, 2.0)), ValueError),
                      (lambda: N.newton_schulz(G, coefficients=(50.0, 0.0, 0.0)), ValueError),
                      (lambda: N.newton_schulz(G, eps=-1.0), ValueError),
                      (lambda: N.Muon([torch.nn.Parameter(G[0])]), ValueError),
                      (lambda: N.Muon([torch.nn.Parameter(G)], momentum=1.0), ValueError)]:
        with pytest.raises(err):
            call()


def test_muon_steps():
    """Three steps on parameters of two shapes (one of them twice: a batch) against the step in 64 bits."""
    from lookatmyquant_b200 import orthogonal as N
    params = [torch.nn.Parameter(update(*s, seed=i)) for i, s in enumerate([(64, 96), (200, 48), (64, 96)])]
    opt = N.Muon(params, lr=0.1, momentum=0.9, weight_decay=0.01)
    ref = [p.detach().double() for p in params]
    buf = [torch.zeros_like(r) for r in ref]
    moved = [0.0] * 3
    for step in range(3):
        for i, p in enumerate(params):
            p.grad = update(*p.shape, seed=100 * step + i)
        opt.step()
        for i, p in enumerate(params):
            g = p.grad.double()
            buf[i] = 0.9 * buf[i] + g
            rate = 0.1 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
            O = exact(g + 0.9 * buf[i])
            ref[i] = ref[i] * (1 - 0.1 * 0.01) - rate * O
            moved[i] += rate * float(O.norm())
            # momentum in fp32: its rounding moves small singular values a little more than the products do
            assert float((p.detach().double() - ref[i]).norm()) <= 1.1 * TOL * moved[i]
