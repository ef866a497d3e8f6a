"""Attention forwards and backwards against the formulas in 64 bits.

Tolerances, element by element, from the arithmetic alone (u = 2^-8, bf16's unit roundoff). The operands are bf16 and
enter exactly; S, the softmax and every accumulation are fp32 (their errors, some 2^-16 of the terms' magnitudes at
most, are the factor 1.05 and the 2^-16 terms below); P and dS are rounded to bf16 once before the second product and
each output once:
  O    : u·(|O| + P·|V|)
  lse  : fp32: 2^-23·(D + 32)·max|scale·q||k| + 2^-20·max(1, |lse|)
  dV   : u·(|dV| + Pᵀ·|dO|)
  dQ   : u·(|dQ| + scale·|dS|·|K|) + scale·(P∘δ)·|K|     δ_i = Σ_d |dO|·tol(O): D is formed from the rounded O
  dK   : u·(|dK| + scale·|dS|ᵀ·|Q|) + scale·(P∘δ)ᵀ·|Q|
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0**-8


def heads(B, H, L, D, g, spread=1.0):
    return (spread * torch.randn(B, L, H, D, device="cuda", generator=g)).bfloat16().transpose(1, 2)


def allowed(B, Lq, Lk, causal, start=None, end=None):
    j = torch.arange(Lk, device="cuda")
    ok = torch.ones(B, 1, Lq, Lk, dtype=torch.bool, device="cuda")
    if causal:
        ok = ok & (j <= torch.arange(Lq, device="cuda")[:, None] + Lk - Lq)
    if start is not None:
        ok = ok & (j >= start.long()[:, None])[:, None, None, :]
    if end is not None:
        ok = ok & (j < end.long()[:, None])[:, None, None, :]
    return ok


def exact(q, k, v, do, scale, ok):
    """Everything in 64 bits, with the tolerances of the docstring."""
    B, Hq, Lq, D = q.shape
    Hkv, Lk = k.shape[1:3]
    G = Hq // Hkv if Hkv else 1
    # what no allowed pair touches must not matter: zero it
    kv_live = ok.any(2).any(1)[:, None, :, None]
    q_live = ok.any(3)[..., None]
    q = torch.where(q_live, q.double(), 0.0)
    k = torch.where(kv_live, k.double(), 0.0).repeat_interleave(G, 1)
    v = torch.where(kv_live, v.double(), 0.0).repeat_interleave(G, 1)
    S = (q @ k.mT * scale).masked_fill(~ok, -math.inf)
    lse = torch.logsumexp(S, -1) if Lk else torch.full((B, Hq, Lq), -math.inf, dtype=torch.float64, device=q.device)
    P = torch.where(ok, (S - torch.where(lse == -math.inf, 0.0, lse)[..., None]).exp(), 0.0)
    o = P @ v
    t = {"o": 1.05 * U * (o.abs() + P @ v.abs()) + 1e-30,
         "lse": 2.0**-23 * (D + 32) * (q.abs() @ k.abs().mT * scale).amax(-1) if Lk else torch.zeros_like(lse)}
    t["lse"] = t["lse"] + 2.0**-20 * torch.where(lse == -math.inf, 0.0, lse).abs().clamp(min=1.0)
    out = {"o": o, "lse": lse}
    if do is not None:
        do = torch.where(q_live, do.double(), 0.0)
        fold = lambda x: x.reshape(B, Hkv, G, *x.shape[2:]).sum(2)
        dP = do @ v.mT
        dS = P * (dP - (P * dP).sum(-1, keepdim=True))
        out["dq"], out["dk"], out["dv"] = dS @ k * scale, fold(dS.mT @ q) * scale, fold(P.mT @ do)
        delta = (do.abs() * t["o"]).sum(-1, keepdim=True)
        loose = P * (delta + 2.0**-16 * (do.abs() @ v.abs().mT))
        t["dv"] = 1.05 * U * (out["dv"].abs() + fold(P.mT @ do.abs())) + 1e-30
        t["dq"] = 1.05 * U * (out["dq"].abs() + scale * dS.abs() @ k.abs()) + scale * loose @ k.abs() + 1e-30
        t["dk"] = (1.05 * U * (out["dk"].abs() + scale * fold(dS.abs().mT @ q.abs())) + scale * fold(loose.mT @ q.abs())
                   + 1e-30)
    return out, t


def check(got, want, tol):
    for name, x in got.items():
        w, t = want[name], tol[name]
        assert x.shape == w.shape, name
        inf = w == -math.inf
        assert torch.equal(x == -math.inf, inf), name
        assert bool(x[~inf].isfinite().all()), name
        over = ((x.double() - w).abs() > t) & ~inf
        assert not bool(over.any()), (name, int(over.sum()), float((x.double() - w)[over].abs().max()))


def both(q, k, v, do, causal, start=None, end=None, scale=None):
    from lookatmyquant_b200 import attention as A
    o, lse = A.forward(q, k, v, scale, causal, start, end)
    dq, dk, dv = A.backward(do, q, k, v, o, lse, scale, causal, start, end)
    A.check_status()
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


SHAPES = [  # B, Hq, Hkv, Lq, Lk, D
    (1, 1, 1, 1, 1, 64), (2, 3, 1, 2, 2, 128), (1, 2, 2, 17, 17, 8), (1, 3, 1, 77, 77, 64), (2, 4, 2, 127, 127, 40),
    (1, 2, 1, 128, 128, 128), (1, 2, 1, 129, 129, 128), (2, 3, 3, 256, 256, 96), (1, 6, 2, 257, 257, 64),
    (1, 2, 2, 385, 385, 80), (3, 8, 1, 300, 300, 128), (1, 2, 1, 1, 700, 128), (1, 4, 2, 5, 1000, 64),
    (2, 2, 1, 130, 517, 128), (1, 2, 2, 513, 129, 64), (1, 3, 1, 200, 3, 128), (1, 15, 5, 1100, 1100, 64),
    (1, 2, 1, 1, 1, 128), (1, 1, 1, 640, 640, 72),
    # few tiles: their work is split over a cluster, by query heads (groups of every kind) and by keys
    (1, 16, 1, 260, 260, 64), (1, 7, 1, 200, 333, 128), (1, 11, 1, 140, 140, 64), (2, 12, 2, 130, 130, 96),
    (1, 2, 1, 3, 1500, 64), (1, 1, 1, 1, 2048, 128), (1, 2, 2, 300, 1290, 128), (1, 1, 1, 129, 640, 40)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,Hq,Hkv,Lq,Lk,D", SHAPES)
def test_forward_and_backward(B, Hq, Hkv, Lq, Lk, D, causal):
    g = torch.Generator("cuda").manual_seed(Lq * 1000 + Lk + D)
    q, k, v, do = (heads(B, H, L, D, g) for H, L in ((Hq, Lq), (Hkv, Lk), (Hkv, Lk), (Hq, Lq)))
    want, tol = exact(q, k, v, do, D ** -0.5, allowed(B, Lq, Lk, causal))
    check(both(q, k, v, do, causal), want, tol)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Lq,Lk", [(150, 150), (300, 300), (40, 290), (290, 260)])
@pytest.mark.parametrize("D", [64, 128])
def test_key_ranges_and_what_masked_places_hold(Lq, Lk, D, causal):
    """Texts of every kind of range: whole, left- and right-padded, inside a tile, one key, none, bounds outside. Keys
    out of range, and queries that see none, hold NaN and infinities (with their gradients): nothing of them arrives."""
    ranges = [(0, Lk), (37, Lk), (0, Lk - 41), (130, 131), (50, 50), (-5, Lk + 9), (Lk - 1, Lk), (129, Lk), (90, 20)]
    start, end = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in zip(*ranges))
    B, Hq, Hkv = len(ranges), 4, 2
    g = torch.Generator("cuda").manual_seed(Lq + Lk + D)
    q, k, v, do = (heads(B, H, L, D, g) for H, L in ((Hq, Lq), (Hkv, Lk), (Hkv, Lk), (Hq, Lq)))
    ok = allowed(B, Lq, Lk, causal, start, end)
    want, tol = exact(q, k, v, do, D ** -0.5, ok)
    clean = both(q, k, v, do, causal, start, end)
    check(clean, want, tol)
    dead_k, dead_q = ~ok.any(2).any(1), ~ok.any(3)[:, 0]
    # a key inside the range that the causal mask keeps from every query is zero work, not garbage: leave it finite
    j = torch.arange(Lk, device="cuda")
    dead_k &= ~((j >= start[:, None]) & (j < end[:, None]))
    for x, dead in ((k, dead_k), (v, dead_k), (q, dead_q), (do, dead_q)):
        rows = x.transpose(1, 2)
        rows[dead] = torch.tensor([math.nan, math.inf, -math.inf, 3e38], device="cuda").repeat(D // 4).bfloat16()
    dirty = both(q, k, v, do, causal, start, end)
    for name in clean:
        assert torch.equal(dirty[name], clean[name]), name
    for name in ("dk", "dv"):
        assert float(dirty[name].transpose(1, 2)[dead_k].abs().sum()) == 0
    assert float(dirty["o"].transpose(1, 2)[dead_q].abs().sum()) == 0
    assert bool((dirty["lse"].transpose(1, 2)[dead_q] == -math.inf).all())


@pytest.mark.parametrize("D", [64, 128])
def test_large_scores(D):
    """Scores of some hundreds, growing and falling along the keys: the running maximum moves, weights underflow."""
    g = torch.Generator("cuda").manual_seed(D)
    L = 400
    q, k, v, do = (heads(1, 2, L, D, g, s) for s in (8.0, 8.0, 1.0, 1.0))
    k *= torch.linspace(0.1, 3.0, L, device="cuda")[:, None].bfloat16()
    for flip in (False, True):
        kk = k.flip(2) if flip else k
        want, tol = exact(q, kk, v, do, D ** -0.5, allowed(1, L, L, False))
        got = both(q, kk, v, do, False)
        # scores of some hundreds in fp32: an error of 2^-23·(D + 32)·|scale·q||k| in the exponent scales P
        e = 2.0**-23 * (D + 32) * float((q.double().abs() @ kk.double().abs().mT).max()) * D ** -0.5
        assert e < 0.05  # first order in e is enough
        grow = {n: t + 3 * e * (t / U) for n, t in tol.items() if n != "lse"}
        check(got, want, {**grow, "lse": tol["lse"]})


def test_scale_and_memory_orders():
    """Tensors of other strides are read in place or copied, with the same result; outputs are projections' order."""
    from lookatmyquant_b200 import attention as A
    g = torch.Generator("cuda").manual_seed(5)
    B, Hq, Hkv, L, D = 2, 4, 2, 200, 64
    q, k, v, do = (heads(B, H, L, D, g) for H in (Hq, Hkv, Hkv, Hq))
    want = both(q, k, v, do, True, scale=0.3)
    w, tol = exact(q, k, v, do, 0.3, allowed(B, L, L, True))
    check(want, w, tol)
    assert want["o"].transpose(1, 2).is_contiguous() and want["dk"].transpose(1, 2).is_contiguous()
    wide = torch.zeros(B, L + 3, Hkv, D + 24, dtype=torch.bfloat16, device="cuda")
    odd = torch.zeros(B, Hkv, L, D + 1, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:, :, 8:8 + D] = k.transpose(1, 2)
    odd[..., 1:] = v
    for kk, vv, qq in ((wide[:, 3:, :, 8:8 + D].transpose(1, 2), odd[..., 1:], q.contiguous()),
                       (k.contiguous(), v.mT.contiguous().mT, q)):
        got = both(qq, kk, vv, do, True, scale=0.3)
        for name in want:
            assert torch.equal(got[name], want[name]), name
    one = torch.ones(1, 1, 1, 1, dtype=torch.bfloat16, device="cuda").expand(B, Hq, L, D)
    o, lse = A.forward(q, k, v)
    for a, b in zip(A.backward(one, q, k, v, o, lse), A.backward(one.contiguous(), q, k, v, o, lse)):
        assert torch.equal(a, b)


def test_equal_calls_give_equal_bits_on_any_stream():
    g = torch.Generator("cuda").manual_seed(6)
    q, k, v, do = (heads(2, H, 700, 128, g) for H in (8, 2, 2, 8))
    want = both(q, k, v, do, True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s):
            got = both(q, k, v, do, True)
        s.synchronize()
        for name in want:
            assert torch.equal(got[name], want[name]), name


def test_gradient_against_differences():
    """The loss Σ c·O in 64 bits, differenced along random directions of q, k and v, against the kernels' gradients:
    within the gradients' own tolerance along the direction, plus the quotient's second-order error."""
    g = torch.Generator("cuda").manual_seed(7)
    B, Hq, Hkv, Lq, Lk, D = 1, 4, 2, 60, 90, 32
    q, k, v, c = (heads(B, H, L, D, g) for H, L in ((Hq, Lq), (Hkv, Lk), (Hkv, Lk), (Hq, Lq)))
    ok = allowed(B, Lq, Lk, True)
    got = both(q, k, v, c, True)
    _, tol = exact(q, k, v, c, D ** -0.5, ok)

    def loss(a, b, d):
        S = (a @ b.repeat_interleave(2, 1).mT * D ** -0.5).masked_fill(~ok, -math.inf)
        return float((torch.softmax(S, -1) @ d.repeat_interleave(2, 1) * c.double()).sum())
    at = [x.double() for x in (q, k, v)]
    for n, name in enumerate(("dq", "dk", "dv")):
        for _ in range(3):
            d = torch.randn(at[n].shape, dtype=torch.float64, device="cuda", generator=g)
            h = 1e-4
            up, dn = list(at), list(at)
            up[n], dn[n] = at[n] + h * d, at[n] - h * d
            quotient = (loss(*up) - loss(*dn)) / (2 * h)
            bound = float((tol[name] * d.abs()).sum()) + 1e-3
            assert abs(quotient - float((got[name].double() * d).sum())) <= bound


def test_offsets_past_32_bits():
    """Keys beyond 2^31 elements (2^32 bytes) of their tensors: the last 300 of 2.2 million, and their gradients."""
    B, Hq, Hkv, Lq, Lk, D, used = 1, 8, 8, 70, 2_200_000, 128, 300
    g = torch.Generator("cuda").manual_seed(9)
    k = torch.zeros(B, Lk, Hkv, D, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    v = torch.zeros_like(k)
    q, do, tail_k, tail_v = (heads(B, H, L, D, g) for H, L in ((Hq, Lq), (Hq, Lq), (Hkv, used), (Hkv, used)))
    k[:, :, -used:], v[:, :, -used:] = tail_k, tail_v
    start = torch.tensor([Lk - used], dtype=torch.int32, device="cuda")
    got = both(q, k, v, do, False, start, None)
    want, tol = exact(q, tail_k, tail_v, do, D ** -0.5, allowed(B, Lq, used, False))
    for name in ("dk", "dv"):
        assert not bool(got[name][:, :, :-used].any())
        got[name] = got[name][:, :, -used:]
    check(got, want, tol)


def test_no_queries_or_no_keys():
    from lookatmyquant_b200 import attention as A
    e = lambda H, L: torch.randn(2, H, L, 64, device="cuda").bfloat16()
    o, lse = A.forward(e(4, 9), e(2, 0), e(2, 0))
    assert float(o.abs().sum()) == 0 and bool((lse == -math.inf).all())
    dq, dk, dv = A.backward(e(4, 9), e(4, 9), e(2, 0), e(2, 0), o, lse)
    assert float(dq.abs().sum()) == 0 and dk.shape == dv.shape == (2, 2, 0, 64)
    o, lse = A.forward(e(4, 0), e(2, 9), e(2, 9))
    assert o.shape == (2, 4, 0, 64) and lse.shape == (2, 4, 0)
    dq, dk, dv = A.backward(e(4, 0), e(4, 0), e(2, 9), e(2, 9), o, lse)
    assert dq.shape == (2, 4, 0, 64) and float(dk.abs().sum()) == float(dv.abs().sum()) == 0
    z = torch.zeros(0, 4, 5, 64, dtype=torch.bfloat16, device="cuda")
    assert A.forward(z, z, z)[0].shape == (0, 4, 5, 64)
    A.check_status()


def test_autograd():
    from lookatmyquant_b200 import attention as A
    g = torch.Generator("cuda").manual_seed(8)
    q, k, v, do = (heads(1, H, 150, 64, g) for H in (6, 2, 2, 6))
    want = both(q, k, v, do, True)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    A.attention(*leaves).backward(do)
    for x, name in zip(leaves, ("dq", "dk", "dv")):
        assert torch.equal(x.grad, want[name])


def test_refusals():
    from lookatmyquant_b200 import attention as A
    t = lambda *s, dt=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dt)
    q, k = t(2, 4, 9, 64), t(2, 2, 9, 64)
    o, lse = A.forward(q, k, k)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")
    for call, err in [(lambda: A.forward(q.float(), k, k), TypeError), (lambda: A.forward(q.cpu(), k, k), TypeError),
                      (lambda: A.forward(q[0], k, k), ValueError), (lambda: A.forward(q, k, k[:, :1]), ValueError),
                      (lambda: A.forward(q, t(2, 3, 9, 64), t(2, 3, 9, 64)), ValueError),
                      (lambda: A.forward(t(2, 4, 9, 12), t(2, 2, 9, 12), t(2, 2, 9, 12)), ValueError),
                      (lambda: A.forward(t(2, 4, 9, 136), t(2, 2, 9, 136), t(2, 2, 9, 136)), ValueError),
                      (lambda: A.forward(q, k, k, scale=0.0), ValueError),
                      (lambda: A.forward(q, k, k, scale=math.inf), ValueError),
                      (lambda: A.forward(q, k, k, scale=math.nan), ValueError),
                      (lambda: A.forward(q, k, k, key_end=i32(3)), ValueError),
                      (lambda: A.forward(q, k, k, key_end=i32(2).long()), ValueError),
                      (lambda: A.backward(q, q, k, k, o[:, :2], lse), ValueError),
                      (lambda: A.backward(q, q, k, k, o, lse[..., :1]), ValueError),
                      (lambda: A.backward(q.float(), q, k, k, o, lse), TypeError),
                      (lambda: A.backward(q, q, k, k, o, lse.double()), ValueError)]:
        with pytest.raises(err):
            call()
