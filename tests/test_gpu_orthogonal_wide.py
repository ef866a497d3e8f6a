"""Newton-Schulz in tiles of 256 x 256 on pairs of CTAs against the iteration in 64 bits: several tiles a pair and mirrored
ones, tall and wide, remainders of every kind, batches, many slices of K, all of them with Muon's tolerance (the bf16
output's rounding, at most 2^-8 of each entry and uniform, and ten roundings of 2^-11)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
MUON = (3.4445, -4.7750, 2.0315)
TOL = math.hypot(2.0**-8, 10 * 2.0**-11) / math.sqrt(3)


def exact(G, coefficients):
    X = G.double()
    X = X / (torch.linalg.matrix_norm(X, keepdim=True) + 1e-7)
    tall = X.shape[-2] > X.shape[-1]
    X = X.mT if tall else X
    for a, b, c in coefficients:
        A = X @ X.mT
        X = a * X + (b * A + c * A @ A) @ X
    return X.mT if tall else X


def update(*shape, seed=0, rank=6):
    g = torch.Generator("cuda").manual_seed(seed)
    m, n = shape[-2:]
    G = torch.randn(*shape[:-2], m, rank, device="cuda", generator=g) @ torch.randn(*shape[:-2], rank, n, device="cuda",
                                                                                   generator=g)
    return 1e-3 * (G + torch.randn(*shape, device="cuda", generator=g)) * torch.exp(
        0.5 * torch.randn(*shape[:-1], 1, device="cuda", generator=g))


def check(G, coefficients=(MUON,) * 5):
    from lookatmyquant_b200 import orthogonal as N
    got, want = N.newton_schulz(G, steps=len(coefficients), coefficients=coefficients), exact(G, coefficients)
    assert got.shape == want.shape and got.dtype == torch.bfloat16
    err, norm = (torch.linalg.matrix_norm(x) for x in (got.double() - want, want))
    assert bool((err <= TOL * norm).all()), float((err / norm).max())
    # no tile, row or column of it worse than the rest: an entry that was left out is off by itself
    off = (got.double() - want).abs()
    assert bool((off <= 2.0**-8 * want.abs() + 12 * TOL * norm[..., None, None] / math.sqrt(G.shape[-1] * G.shape[-2])).all())
    assert torch.equal(got, N.newton_schulz(G, steps=len(coefficients), coefficients=coefficients))
    N.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", [(2305, 2049), (2049, 2305), (2304, 2304), (1999, 2560), (2560, 2175), (1030, 4100),
                                 (4100, 1030), (513, 8200), (8200, 513)])
def test_matrices(m, n, dtype):
    check(update(m, n, seed=m + n).to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,m,n", [(19, 300, 513), (19, 513, 300), (40, 257, 256), (40, 255, 500), (80, 130, 200),
                                   (13, 769, 520)])
def test_batches(b, m, n, dtype):
    G = update(b, m, n, seed=b) * torch.logspace(-3, 3, b, device="cuda")[:, None, None]
    check(G.to(dtype))


@pytest.mark.parametrize("m,n", [(2305, 2049), (2049, 2305)])
@pytest.mark.parametrize("steps", [1, 2, 7])
def test_steps(m, n, steps):
    check(update(m, n, seed=steps), (MUON,) * steps)


@pytest.mark.parametrize("m,n", [(2305, 2049), (2049, 2305)])
def test_three_products_everywhere(m, n):
    check(update(m, n, seed=9), ((8.28721201814563, -23.595886519098837, 17.300387312530933),
                                 (4.107059111542203, -2.9478499167379106, 0.5448431082926601),
                                 (3.9486908534822946, -2.908902115962949, 0.5518191394370137),
                                 (3.3184196573706015, -2.488488024314874, 0.51004894012372),
                                 (2.300652019954817, -1.6689039845747493, 0.4188073119525673)))


@pytest.mark.parametrize("m,n", [(2305, 2049), (2049, 2305)])
def test_strided_updates_and_non_finite_ones(m, n):
    from lookatmyquant_b200 import orthogonal as N
    big = update(m + 3, n + 70, seed=11)
    want = N.newton_schulz(big[2:m + 2, 9:n + 9].contiguous())
    assert torch.equal(N.newton_schulz(big[2:m + 2, 9:n + 9]), want)
    for bad in (math.nan, math.inf):
        G = big[:m, :n].clone()
        G[m // 2, n // 3] = bad
        assert bool(N.newton_schulz(G).isnan().all())
