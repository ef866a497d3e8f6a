"""The scaled embedding lookup and its gradient against 64-bit sums.

Tolerances, from the arithmetic alone (u the output type's unit roundoff: 2^-24 fp32, 2^-8 bf16):
lookup: one fp32 product, rounded to the type: |err| <= (u + 2^-24)·|y|.
gradient: c terms added in fp32 in some fixed order, one product, one rounding: |err| <= (c + 1)·2^-24·scale·Σ|dy| + u·|dE|
(and u·|old| + 2^-24·(...) more when added to an existing gradient)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}


def zipf_ids(n, V, g, s=1.1):
    w = torch.arange(1, V + 1, dtype=torch.float64).pow(-s)
    perm = torch.randperm(V, generator=g)
    return perm[torch.multinomial(w, n, replacement=True, generator=g)] if n else torch.zeros(0, dtype=torch.long)


def check_gradient(got, dy, ids, V, scale, padding, old=None):
    dt = dy.dtype
    keep = torch.ones_like(ids, dtype=torch.bool) if padding is None else ids != padding
    keep &= (ids >= 0) & (ids < V)
    i, x = ids[keep], dy.double()[keep]
    want = torch.zeros(V, dy.shape[-1], dtype=torch.float64, device=dy.device).index_add_(0, i, x) * scale
    mags = torch.zeros_like(want).index_add_(0, i, x.abs()) * abs(scale)
    c = torch.bincount(i, minlength=V).double()[:, None]
    tol = (c + 2) * 2.0**-24 * mags
    if old is not None:
        want = want + old.double()
        tol = tol + 2.0**-24 * want.abs()
    tol = tol + U[dt] * want.abs() * (1 + 1e-6)
    assert got.shape == want.shape and got.dtype == dt
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,d,n", [(1, 8, 1), (5, 1, 3), (100, 7, 33), (1000, 64, 257), (300, 1000, 2049),
                                   (49152, 960, 500), (513, 2560, 64)])
def test_lookup(V, d, n, dtype):
    from lookatmyquant_b200 import embedding as E
    g = torch.Generator().manual_seed(V + d + n)
    table = torch.randn(V, d, generator=g).to(dtype).cuda()
    ids = zipf_ids(n, V, g).cuda()
    scale = math.sqrt(d)
    y = E.lookup(table, ids, scale)
    want = table.double()[ids] * scale
    assert bool(((y.double() - want).abs() <= (U[dtype] + 2.0**-24) * (1 + 1e-6) * want.abs()).all())
    assert torch.equal(y, (table[ids].float() * torch.tensor(scale, dtype=torch.float32)).to(dtype))
    assert torch.equal(E.lookup(table, ids.int(), scale), y)
    pad = int(ids[0])
    yp = E.lookup(table, ids.reshape(1, -1), scale, padding_idx=pad)
    assert yp.shape == (1, n, d)
    assert bool((yp[0][ids == pad] == 0).all()) and torch.equal(yp[0][ids != pad], y[ids != pad])
    E.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,d,n,s", [(1, 8, 1, 1.1), (1, 8, 5000, 1.1), (5, 1, 3, 1.1), (100, 7, 33, 1.1),
                                     (1000, 64, 257, 1.1), (300, 1000, 2049, 1.1), (49152, 960, 4097, 1.1),
                                     (131072, 64, 20000, 1.1), (2, 320, 3000, 1.1), (70000, 2560, 300, 0.0),
                                     (255, 40, 65536, 1.1), (256, 40, 8192, 2.0), (4000000, 8, 1000, 0.5)])
def test_gradient(V, d, n, s, dtype):
    from lookatmyquant_b200 import embedding as E
    g = torch.Generator().manual_seed(V + d + n)
    ids = zipf_ids(n, V, g, s).cuda()
    dy = torch.randn(n, d, generator=g).to(dtype).cuda()
    scale = math.sqrt(d)
    got = E.lookup_gradient(dy, ids, V, scale)
    check_gradient(got, dy, ids, V, scale, None)
    assert torch.equal(got, E.lookup_gradient(dy, ids.int(), V, scale))  # and equal bits on a second call
    pad = int(ids[n // 2])
    check_gradient(E.lookup_gradient(dy, ids, V, scale, padding_idx=pad), dy, ids, V, scale, pad)
    old = torch.randn(V, d, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(dtype)
    into = old.clone()
    assert E.lookup_gradient(dy, ids, V, scale, padding_idx=pad, out=into) is into
    check_gradient(into, dy, ids, V, scale, pad, old)
    E.check_status()


def test_gradient_against_differences():
    """d/dE of Σ c·(lookup) by central differences in 64 bits of the formula equals the kernel's gradient: the lookup is
    linear, so the difference quotient is exact up to rounding."""
    from lookatmyquant_b200 import embedding as E
    g = torch.Generator().manual_seed(3)
    V, d, n, scale = 6, 5, 40, 1.75
    ids = torch.randint(0, V, (n,), generator=g)
    c = torch.randn(n, d, generator=g)
    got = E.lookup_gradient(c.cuda(), ids.cuda(), V, scale).double().cpu()
    table = torch.randn(V, d, generator=g).double()
    f = lambda t: float((t[ids] * scale * c.double()).sum())
    for v in range(V):
        for j in range(d):
            up, dn = table.clone(), table.clone()
            up[v, j] += 0.5
            dn[v, j] -= 0.5
            assert abs(f(up) - f(dn) - float(got[v, j])) <= 42 * 2.0**-24 * scale * float(c.abs().sum())


def test_strided_rows_and_unaligned_pieces():
    from lookatmyquant_b200 import embedding as E
    g = torch.Generator().manual_seed(4)
    for dtype in (torch.float32, torch.bfloat16):
        big = torch.randn(50, 200, generator=g).to(dtype).cuda()
        ids = torch.randint(0, 50, (77,), generator=g).cuda()
        for lo, d in ((0, 64), (8, 64), (3, 64), (1, 9)):
            t = big[:, lo:lo + d]
            assert torch.equal(E.lookup(t, ids, 2.0), E.lookup(t.contiguous(), ids, 2.0))
            dy = torch.randn(77, 200, generator=g).to(dtype).cuda()[:, lo:lo + d]
            want = E.lookup_gradient(dy.contiguous(), ids, 50, 0.5)
            check_gradient(want, dy, ids, 50, 0.5, None)
            assert torch.equal(E.lookup_gradient(dy, ids, 50, 0.5), want)
            into = torch.zeros(50, 200, dtype=dtype, device="cuda")
            E.lookup_gradient(dy, ids, 50, 0.5, out=into[:, lo:lo + d])
            assert torch.equal(into[:, lo:lo + d], want) and float(into[:, lo + d:].abs().sum()) == 0
    assert torch.equal(E.lookup(big.t(), ids % 50, 1.0), big.t()[ids % 50])  # columns of a matrix: copied
    assert torch.equal(E.lookup(big, ids.flip(0)[::2], 1.0), big[ids.flip(0)[::2]])


def test_empty_and_one_token():
    from lookatmyquant_b200 import embedding as E
    t = torch.randn(10, 16, device="cuda")
    none = torch.zeros(0, dtype=torch.long, device="cuda")
    assert E.lookup(t, none).shape == (0, 16)
    assert torch.equal(E.lookup_gradient(torch.zeros(0, 16, device="cuda"), none, 10), torch.zeros(10, 16, device="cuda"))
    one = torch.tensor(7, device="cuda")
    assert torch.equal(E.lookup(t, one), t[7])
    got = E.lookup_gradient(t[7], one, 10, 3.0)
    assert torch.equal(got[7], t[7] * 3.0)
    assert bool((got[torch.arange(10, device="cuda") != 7] == 0).all())
    assert E.lookup_gradient(torch.zeros(0, 16, device="cuda"), none, 0).shape == (0, 16)


def test_non_finite_rows_stay_where_they_are():
    """An infinity or NaN reaches the rows of its own token only, and none from a padding token."""
    from lookatmyquant_b200 import embedding as E
    dy = torch.ones(300, 24, device="cuda")
    ids = torch.arange(300, device="cuda") % 7
    dy[3], dy[4], dy[6] = math.inf, math.nan, math.nan
    got = E.lookup_gradient(dy, ids, 9, padding_idx=6)
    assert bool(got[3].isinf().all()) and bool(got[4].isnan().all())
    assert bool(got[[0, 1, 2, 5, 6, 7, 8]].isfinite().all()) and float(got[6:].abs().sum()) == 0


def test_invalid_ids_are_reported():
    from lookatmyquant_b200 import embedding as E
    t = torch.randn(10, 16, device="cuda")
    E.check_status()
    for bad in (10, -1, 2**40):
        ids = torch.tensor([1, bad, 2], device="cuda")
        y = E.lookup(t, ids)
        assert torch.equal(y[[0, 2]], t[[1, 2]]) and float(y[1].abs().sum()) == 0
        with pytest.raises(ValueError, match="outside the table"):
            E.check_status()
        check_gradient(E.lookup_gradient(t[:3], ids, 10), t[:3], ids, 10, 1.0, None)
        with pytest.raises(ValueError, match="outside the table"):
            E.check_status()
    E.check_status()


def test_refusals():
    from lookatmyquant_b200 import embedding as E
    t, ids = torch.randn(10, 16, device="cuda"), torch.zeros(3, dtype=torch.long, device="cuda")
    for call, err in [(lambda: E.lookup(t.half(), ids), TypeError), (lambda: E.lookup(t.cpu(), ids), TypeError),
                      (lambda: E.lookup(t, ids.float()), TypeError), (lambda: E.lookup(t, ids.cpu()), TypeError),
                      (lambda: E.lookup(t[0], ids), ValueError),
                      (lambda: E.lookup_gradient(t, ids, 10), ValueError),
                      (lambda: E.lookup_gradient(t[:3], ids, -1), ValueError),
                      (lambda: E.lookup_gradient(t[:3], ids, 10, out=t[:9]), ValueError),
                      (lambda: E.lookup_gradient(t[:3], ids, 10, out=t.bfloat16()), ValueError)]:
        with pytest.raises(err):
            call()


def test_another_stream():
    from lookatmyquant_b200 import embedding as E
    g = torch.Generator().manual_seed(9)
    t, ids = torch.randn(5000, 512, generator=g).cuda(), torch.randint(0, 5000, (9000,), generator=g).cuda()
    want_y = E.lookup(t, ids, 2.0)
    want_g = E.lookup_gradient(want_y, ids, 5000, 2.0)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y = E.lookup(t, ids, 2.0)
        gr = E.lookup_gradient(y, ids, 5000, 2.0)
    s.synchronize()
    assert torch.equal(y, want_y) and torch.equal(gr, want_g)


def test_autograd():
    from lookatmyquant_b200 import embedding as E
    g = torch.Generator().manual_seed(11)
    t = torch.randn(40, 24, generator=g).cuda().requires_grad_(True)
    ids = torch.randint(0, 40, (3, 50), generator=g).cuda()
    c = torch.randn(3, 50, 24, generator=g).cuda()
    (E.scaled_embedding(t, ids, 4.0, 0) * c).sum().backward()
    check_gradient(t.grad, c.reshape(-1, 24), ids.reshape(-1), 40, 4.0, 0)


def test_offsets_past_32_bits():
    """Rows that lie beyond 2^31 elements (2^32 bytes) of the table, of the gradient and of the tokens' rows."""
    from lookatmyquant_b200 import embedding as E
    V, d = 2_200_000, 1024
    table = torch.zeros(V, d, dtype=torch.bfloat16, device="cuda")
    rows = torch.tensor([0, V // 2, V - 2, V - 1], device="cuda")
    g = torch.Generator("cuda").manual_seed(1)
    table[rows] = torch.randn(4, d, device="cuda", generator=g).bfloat16()
    ids = rows[torch.randint(0, 4, (3000,), device="cuda", generator=g)]
    assert torch.equal(E.lookup(table, ids, 2.0), table[ids] * 2)
    dy = torch.randn(3000, d, device="cuda", generator=g).bfloat16()
    for n in (1000, 3000):  # both ways to the gradient
        dE = E.lookup_gradient(dy[:n], ids[:n], V, 0.5)
        for r in rows:
            mine = dy[:n][ids[:n] == r].double()
            tol = (len(mine) + 2) * 2.0**-24 * 0.5 * mine.abs().sum(0) + 2.0**-8 * 0.5 * mine.sum(0).abs() * (1 + 1e-6)
            assert bool(((dE[r].double() - 0.5 * mine.sum(0)).abs() <= tol).all())
        dE[rows] = 0
        assert not bool(dE.any())
    E.check_status()
