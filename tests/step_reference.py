"""Plain 64-bit forms of the norms around a block, each value with a bound on what fp32 arithmetic may be off by.

`e` is the bound on a value before its last rounding. K counts the roundings of a row's sum: up to 32 products in a thread, 5
shuffles, 16 warps, and some around it; S those of a sum over rows: the rows of a range, the teams of a block and the blocks.
"""

import torch

F32 = 2.0**-24  # half a step of fp32
K, S = 64, 700


def half(dtype):
    return torch.finfo(dtype).eps / 2


def mean(x):
    return x.mean(-1, keepdim=True)


def unit(x, ex, eps):
    """(x·r, its error, r): x̂ of a row whose elements are off by ex."""
    ms = mean(x * x)
    r = (ms + eps).rsqrt()
    rel = K * F32 + mean(ex * x.abs()) * r * r  # of r
    return x * r, (ex + x.abs() * rel) * r * 1.01, r


def join_forward(residual, branch, weight=None, post=None, gate=None, scale=1.0, eps=1e-6, offset=0.0):
    """((h, error), (y, error) or None), y from the unrounded h."""
    b, eb = branch.double(), torch.zeros_like(branch, dtype=torch.float64)
    if post is not None:
        u = post.double() + offset
        b, eb, _ = unit(b, eb, eps)
        b, eb = b * u, eb * u.abs() + 2 * F32 * (b * u).abs()
    if gate is not None:
        g = gate.double()
        b, eb = b * g, eb * g.abs() + F32 * (b * g).abs()
    h = residual.double() + scale * b
    eh = abs(scale) * (eb + F32 * b.abs()) + F32 * h.abs()
    if weight is None:
        return (h, eh), None
    return (h, eh), norm_forward(h, weight, eps, offset, eh)


def norm_forward(x, weight, eps=1e-6, offset=0.0, ex=None):
    x = x.double()
    w = weight.double() + offset
    n, en, _ = unit(x, torch.zeros_like(x) if ex is None else ex, eps)
    return n * w, en * w.abs() + 3 * F32 * (n * w).abs()


def norm_gradient(dy, ey, x, weight, eps, offset):
    """((dx, error), (dweight, error)): dy off by ey."""
    n, en, r = unit(x, torch.zeros_like(x), eps)
    w = weight.double() + offset
    t, et = dy * w, ey * w.abs() + 2 * F32 * (dy * w).abs()
    c = mean(t * n)
    ec = mean(et * n.abs() + t.abs() * en) + K * F32 * mean((t * n).abs())
    dx = r * (t - n * c)
    edx = r * (et + en * c.abs() + n.abs() * ec + 3 * F32 * (t.abs() + (n * c).abs())) + K * F32 * dx.abs()
    rows = tuple(range(x.ndim - 1))
    dw = (dy * n).sum(rows)
    edw = (ey * n.abs() + dy.abs() * en).sum(rows) + (S * F32) * (dy * n).abs().sum(rows)
    return (dx, edx), (dw, edw)


def join_backward(dh, dy, h, branch, weight=None, post=None, gate=None, scale=1.0, eps=1e-6, offset=0.0):
    """{"residual", "branch", "weight", "post", "gate"}: (gradient, error) of those there are."""
    h, b = h.double(), branch.double()
    zero = torch.zeros_like(h)
    g, eg = (zero, zero) if dh is None else (dh.double(), zero)
    out = {}
    if weight is not None:
        (dn, edn), out["weight"] = norm_gradient(zero if dy is None else dy.double(), zero, h, weight, eps, offset)
        g = g + dn
        eg = edn + F32 * g.abs()
    out["residual"] = (g, eg)
    t, et = scale * g, abs(scale) * eg + F32 * (scale * g).abs()
    if gate is not None:
        p, ep = b, zero
        if post is not None:
            u = post.double() + offset
            p, ep, _ = unit(b, zero, eps)
            p, ep = p * u, ep * u.abs() + 2 * F32 * (p * u).abs()
        dg, edg = t * p, et * p.abs() + t.abs() * ep + F32 * (t * p).abs()
        full = (1,) * (b.ndim - gate.ndim) + tuple(gate.shape)
        shared = tuple(i for i, n in enumerate(full) if n != b.shape[i])
        if shared:
            edg = edg.sum(shared, keepdim=True) + (S * F32) * dg.abs().sum(shared, keepdim=True)
            dg = dg.sum(shared, keepdim=True)
        out["gate"] = dg.reshape(gate.shape), edg.reshape(gate.shape)
        t, et = t * gate.double(), et * gate.double().abs() + F32 * (t * gate.double()).abs()
    if post is not None:
        (t, et), out["post"] = norm_gradient(t, et, b, post, eps, offset)
    out["branch"] = (t, et)
    return out


def assert_close(got, want, what=""):
    """Within the error of the value and one rounding to got's type (and its smallest number)."""
    value, error = want
    assert got.shape == value.shape, (what, got.shape, value.shape)
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    allowed = error + half(got.dtype) * (value.abs() + error) + tiny
    off = (got.double() - value).abs()
    worst = (off / allowed.clamp_min(1e-300)).max() if off.numel() else torch.zeros(())
    assert bool((off <= allowed).all()), f"{what}: {float(worst):.3f} times the allowed error"
