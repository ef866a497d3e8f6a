"""The norms around a block against their 64-bit forms, with the errors that fp32 arithmetic and one rounding allow."""

import pytest
import torch
from step_reference import assert_close, join_backward, join_forward, norm_forward, norm_gradient

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def N():
    from lookatmyquant_b200 import norms
    return norms


def generator(seed):
    return torch.Generator("cuda").manual_seed(seed)


def values(g, *shape, scale=1.0, dtype=FP):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


WIDTHS = [1, 2, 7, 8, 31, 32, 33, 64, 96, 128, 129, 256, 257, 960, 1000, 1337, 2560, 4096, 4097, 4104, 8192, 8200, 9728, 16383, 16384]


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_norm(N, d, dtype):
    for n in (1, 3, 77, 700):
        g = generator(d + n)
        x = values(g, n, d, scale=torch.exp(torch.randn(d, device="cuda", generator=g)), dtype=dtype)
        w, dy = values(g, d, dtype=dtype), values(g, n, d, scale=1e-3, dtype=dtype)
        assert_close(N.norm_forward(x, w, eps=1e-5, offset=1.0), norm_forward(x, w, 1e-5, 1.0), f"y of {n}")
        dx, dw = N.norm_backward(dy, x, w, eps=1e-5, offset=1.0)
        wx, ww = norm_gradient(dy.double(), torch.zeros_like(x).double(), x.double(), w, 1e-5, 1.0)
        assert_close(dx, wx, f"dx of {n}")
        assert_close(dw, ww, f"dw of {n}")


def case(seed, n, d, residual, branch, post, gate, pre, texts=1):
    """The tensors of a join over `texts` texts of n rows."""
    g = generator(seed)
    shape = (texts, n, d)
    t = dict(residual=values(g, *shape, dtype=residual), branch=values(g, *shape, scale=0.5, dtype=branch),
             weight=values(g, d, dtype=branch) if pre else None, post=values(g, d, dtype=branch) if post else None, gate=None)
    if gate:
        gates = {"channel": (d,), "one": (1, 1, d), "text": (texts, 1, d), "token": shape}[gate]
        t["gate"] = values(g, *gates, dtype=branch)
    return t


def check_join(N, t, scale=0.3, eps=1e-5, offset=0.0, seed=5):
    args = (t["weight"], t["post"], t["gate"], scale, eps, offset)
    h, y = N.join_forward(t["residual"], t["branch"], *args)
    wh, wy = join_forward(t["residual"], t["branch"], *args)
    assert_close(h, wh, "h")
    if y is not None:
        assert_close(y, wy, "y")
    else:
        assert wy is None
    g = generator(seed)
    dh = values(g, *h.shape, scale=1e-3, dtype=h.dtype)
    dy = None if y is None else values(g, *h.shape, scale=1e-3, dtype=y.dtype)
    got = dict(zip(("residual", "branch", "weight", "post", "gate"), N.join_backward(dh, dy, h, t["branch"], *args)))
    want = join_backward(dh, dy, h, t["branch"], *args)
    assert {k for k, x in got.items() if x is not None} == set(want)
    for k, x in want.items():
        assert_close(got[k], x, f"d_{k}")


@pytest.mark.parametrize("d", [1, 8, 33, 128, 960, 1337, 2560, 4104, 9728, 16383, 16384])
@pytest.mark.parametrize("types", [(BF, BF), (FP, BF), (FP, FP)])
def test_join_of_all_widths_and_types(N, d, types):
    check_join(N, case(d, 77, d, *types, True, "text", True, texts=3))
    check_join(N, case(d, 130, d, *types, False, None, True), scale=1.0)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [None, "channel", "one", "text", "token"])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("n,d,texts", [(1, 960, 1), (1, 64, 40), (2, 200, 700), (333, 48, 5), (2000, 256, 2), (37, 129, 90)])
def test_join_of_all_forms(N, post, gate, pre, n, d, texts):
    check_join(N, case(n + d, n, d, BF, BF, post, gate, pre, texts), offset=1.0 if post else 0.0)


@pytest.mark.parametrize("n,texts", [(1, 3), (3, 500), (8, 2000), (700, 7), (5000, 3), (20000, 1)])
@pytest.mark.parametrize("d", [8, 16, 72])
def test_gates_of_texts_of_any_length(N, n, texts, d):
    """Gate rows that a range of rows holds whole, that cross ranges, and one for everything; weights of another type."""
    t = case(n, n, d, FP, BF, True, "text", True, texts)
    for name in ("weight", "post", "gate"):
        t[name] = t[name].float()
    check_join(N, t)


@pytest.mark.parametrize("n,texts", [(1, 40), (2, 700), (3, 900), (5, 1), (600, 3), (400, 1)])
@pytest.mark.parametrize("d,post", [(4097, True), (4099, False), (8200, True)])
def test_gates_of_texts_in_wide_rows(N, n, texts, d, post):
    check_join(N, case(n + d, n, d, FP, BF, post, "text", True, texts))


def test_rows_at_strides(N):
    """Heads out of a joint projection, transposed and sliced tensors, expanded ones: read where they are, or copied."""
    g = generator(3)
    both = values(g, 2, 50, 12 * 64, dtype=BF)
    w = values(g, 64, dtype=BF)
    heads = both.view(2, 50, 12, 64)[:, :, 2:7]
    for x in (heads, heads[:, ::2], heads.transpose(1, 2), heads[..., ::2].repeat_interleave(2, -1), heads[:1, :1],
              both[:, :, 7:71], both[:, :1, :64].expand(2, 9, 64), heads.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)):
        wide = w[:x.shape[-1]]
        assert torch.equal(N.norm_forward(x, wide), N.norm_forward(x.clone(memory_format=torch.contiguous_format), wide))
        dy = values(g, *x.shape, dtype=BF)
        for a, b in zip(N.norm_backward(dy.transpose(0, 1).contiguous().transpose(0, 1), x, wide),
                        N.norm_backward(dy, x.contiguous(), wide)):
            assert_close(a, (b.double(), 2.0**-7 * b.double().abs() + 1e-6))  # sums over rows in vectors or by elements
    t = case(9, 40, 96, FP, BF, True, "text", True, 3)
    want = N.join_forward(t["residual"], t["branch"], t["weight"], t["post"], t["gate"], 0.3)
    for k in ("residual", "branch", "gate"):
        t[k] = torch.stack([t[k], t[k] + 1], -2)[..., 0, :]
    for k in ("weight", "post"):
        t[k] = torch.stack([t[k], t[k] + 1], -1)[..., 0]
    for a, b in zip(want, N.join_forward(t["residual"], t["branch"], t["weight"], t["post"], t["gate"], 0.3)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("shift", [1, 2, 4])
def test_tensors_that_start_anywhere(N, shift):
    t = case(4, 30, 64, BF, BF, True, "channel", True, 2)
    for k, x in t.items():
        flat = torch.zeros(x.numel() + shift, dtype=x.dtype, device="cuda")
        flat[shift:] = x.flatten()
        t[k] = flat[shift:].view(x.shape)
    check_join(N, t)


@pytest.mark.parametrize("d", [64, 37, 4104, 4097, 9728])
@pytest.mark.parametrize("gate", ["text", "token", "channel"])
def test_what_is_not_wanted_is_none(N, d, gate):
    t = case(6, 20, d, BF, BF, True, gate, True, 3)
    h, y = N.join_forward(t["residual"], t["branch"], t["weight"], t["post"], t["gate"])
    args = (h, t["branch"], t["weight"], t["post"], t["gate"])
    every = N.join_backward(h, y, *args)
    for k, name in enumerate(N.PARAMETERS):
        some = N.join_backward(h, y, *args, want=[name])
        assert torch.equal(some[0], every[0]) and torch.equal(some[1], every[1])
        assert [x is not None for x in some[2:]] == [j == k for j in range(3)] and torch.equal(some[2 + k], every[2 + k])
    none = N.join_backward(h, y, *args, want=())
    assert torch.equal(none[1], every[1]) and none[2:] == (None, None, None)
    # no gradient of h, none of y
    for dh, dy in ((None, y), (h, None), (None, None)):
        got = N.join_backward(dh, dy, *args)
        zero = torch.zeros_like(h)
        for a, b in zip(got, N.join_backward(zero if dh is None else dh, zero if dy is None else dy, *args)):
            assert torch.equal(a, b)


def test_equal_calls_give_equal_bits(N):
    t = case(8, 3000, 320, BF, BF, True, "text", True, 4)
    h, y = N.join_forward(t["residual"], t["branch"], t["weight"], t["post"], t["gate"])
    first = N.join_backward(h, y, h, t["branch"], t["weight"], t["post"], t["gate"])
    for _ in range(5):
        for a, b in zip(first, N.join_backward(h, y, h, t["branch"], t["weight"], t["post"], t["gate"])):
            assert torch.equal(a, b)


def test_empty_shapes(N):
    for shape in ((0, 64), (3, 0), (2, 0, 64), (0,)):
        x, w = torch.zeros(shape, device="cuda"), torch.ones(shape[-1], device="cuda")
        assert N.norm_forward(x, w).shape == x.shape
        dx, dw = N.norm_backward(x, x, w)
        assert dx.shape == x.shape and dw.tolist() == [0.0] * shape[-1]
        h, y = N.join_forward(x, x, w, w, w)
        assert h.shape == y.shape == x.shape
        for a, s in zip(N.join_backward(h, y, h, x, w, w, w), (shape, shape, shape[-1:], shape[-1:], shape[-1:])):
            assert a.shape == torch.Size(s) and float(a.abs().sum()) == 0
    x = torch.randn(64, device="cuda")  # a single row without leading axes
    assert_close(N.norm_forward(x, x), norm_forward(x, x))


def test_rows_at_the_ends_of_fp32(N):
    """Squares that overflow fp32, rows of zeros, tiny rows under their eps; a NaN or an infinity stays in its row."""
    g = generator(2)
    for d in (24, 33, 960, 1337, 9728):
        x = values(g, 6, d)
        x[0] *= 1e30
        x[1] *= 3e37
        x[2] = 0
        x[3] *= 1e-25
        x[4] *= 1e19
        w = values(g, d)
        dy = values(g, 6, d)
        assert_close(N.norm_forward(x, w), norm_forward(x, w))
        dx, dw = N.norm_backward(dy, x, w)
        wx, ww = norm_gradient(dy.double(), torch.zeros_like(x).double(), x.double(), w, 1e-6, 0.0)
        assert_close(dx, wx)
        assert_close(dw, ww)
        clean = N.norm_forward(x, w)
        bad = x.clone()
        bad[1, d // 2], bad[4, 0] = float("nan"), float("inf")
        y = N.norm_forward(bad, w)
        rest = [0, 2, 3, 5]
        assert torch.equal(y[rest], clean[rest]) and bool(y[1].isnan().all())
        assert bool(y[4, 0].isnan()) and float(y[4, 1:].abs().sum()) == 0
        t = dict(residual=torch.zeros_like(x), branch=x, weight=w, post=w, gate=None)
        t["residual"][5] = values(g, d)
        check_join(N, t)


def test_gradients_against_differences(N):
    """Along random directions: the 64-bit loss on both sides of the point, against the kernels' gradients. A central
    difference is off by its step squared times a third derivative; the gradients by their own allowed error."""
    t = {k: x.double() for k, x in case(1, 5, 24, FP, FP, True, "text", True, 2).items()}
    g = generator(9)
    dh, dy = values(g, 2, 5, 24), values(g, 2, 5, 24)

    def loss(p):
        (h, _), (y, _) = join_forward(p["residual"], p["branch"], p["weight"], p["post"], p["gate"], 0.7, 1e-3)
        return float((h * dh).sum() + (y * dy).sum())
    p32 = {k: x.float().requires_grad_(True) for k, x in t.items()}
    h, y = N.join(p32["residual"], p32["branch"], p32["weight"], p32["post"], p32["gate"], 0.7, 1e-3)
    ((h * dh).sum() + (y * dy).sum()).backward()
    for k, x in t.items():
        for _ in range(3):
            v = torch.randn(x.shape, device="cuda", generator=g, dtype=torch.float64)
            step = 1e-4
            slope = (loss({**t, k: x + step * v}) - loss({**t, k: x - step * v})) / (2 * step)
            got = float((p32[k].grad.double() * v).sum())
            size = float((p32[k].grad.double() * v).abs().sum())
            assert abs(got - slope) <= 2.0**-16 * size + 1e-5, k


def test_autograd(N):
    """The functions under autograd return what the plain calls do; what needs no gradient costs none; one derivative only."""
    t = case(12, 40, 128, BF, BF, True, "text", True, 3)
    leaves = {k: x.clone().requires_grad_(True) for k, x in t.items()}
    h, y = N.join(*leaves.values(), 0.5)
    dh, dy = values(generator(1), *h.shape, dtype=BF), values(generator(2), *h.shape, dtype=BF)
    torch.autograd.backward((h, y), (dh, dy))
    want = N.join_backward(dh, dy, h, t["branch"], t["weight"], t["post"], t["gate"], 0.5)
    for x, grad in zip(leaves.values(), want):
        assert torch.equal(x.grad, grad) and not x.grad.requires_grad
    # only y, only h, an output alone
    for pick in (0, 1):
        out = N.join(*leaves.values(), 0.5)[pick]
        got = torch.autograd.grad(out, list(leaves.values()), dy, allow_unused=True)
        want = N.join_backward(dy if pick == 0 else None, dy if pick else None, h, t["branch"], t["weight"], t["post"], t["gate"], 0.5)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    x, w = leaves["residual"], leaves["weight"]
    a, b = torch.autograd.grad(N.norm(x, w), (x, w), dy)
    for u, v in zip((a, b), N.norm_backward(dy, t["residual"], t["weight"])):
        assert torch.equal(u, v)
    a, = torch.autograd.grad(N.norm(x, t["weight"]), x, dy)
    assert torch.equal(a, N.norm_backward(dy, t["residual"], t["weight"])[0])
    first, = torch.autograd.grad(N.norm(x, w), x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivatives"):
        first.float().sum().backward()
    # a plain join: one gradient for both, added up where a leaf is both
    x = t["residual"].clone().requires_grad_(True)
    h, y = N.join(x, x, t["weight"])
    h.backward(dh)
    assert torch.equal(x.grad, dh + dh)


def test_graphs_and_streams_hold_the_norms(N):
    """A captured call replayed on new inputs gives what a call gives, bit for bit; two graphs, replayed in turn on two
    streams, do not meet in a workspace."""
    g = generator(4)
    ts = [case(s, 500, 192, BF, BF, True, "text", True, 3) for s in (1, 2)]

    def call(t):
        h, y = N.join_forward(*t.values(), 0.5)
        return (h, y, *N.join_backward(h, y, h, *list(t.values())[1:], 0.5))
    graphs, outs = [], []
    for t in ts:
        call(t)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(t))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for t in ts:
            for x in t.values():
                x.copy_(values(g, *x.shape))
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for t, out in zip(ts, outs):
            for a, b in zip(out, call(t)):
                assert torch.equal(a, b)


def test_a_captured_training_step(N):
    """Forward and backward under autograd in one graph, replayed on new inputs."""
    x = torch.randn(3, 40, 64, device="cuda").requires_grad_(True)
    w = torch.randn(64, device="cuda").requires_grad_(True)

    def step():
        h, y = N.join(x, torch.sin(x), w, w, None, 0.5)
        return torch.autograd.grad((h * y).sum(), (x, w))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(2):
        with torch.no_grad():
            x.normal_(), w.normal_()
        graph.replay()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_many_rows(N):
    """Offsets behind 2^31 elements, in the last rows."""
    n, d = 140_000, 16384
    x = torch.empty(n, d, dtype=BF, device="cuda")
    x[-3:] = values(generator(1), 3, d, dtype=BF)
    x[:-3] = 0
    w = values(generator(2), d, dtype=BF)
    y = N.norm_forward(x, w)
    assert_close(y[-3:], norm_forward(x[-3:], w, 1e-6))
    assert float(y[1000:1010].abs().sum()) == 0
    dx, dw = N.norm_backward(y, x, w)
    wx, ww = norm_gradient(y[-3:].double(), torch.zeros(3, d, device="cuda").double(), x[-3:].double(), w, 1e-6, 0.0)
    assert_close(dx[-3:], wx)
    assert_close(dw, ww)


def test_another_stream_and_device_context(N):
    """On a stream of its own, beside work on the default one; the results belong to that stream."""
    t = case(3, 300, 256, BF, BF, True, "text", True, 4)
    args = (t["weight"], t["post"], t["gate"], 0.3)
    h, y = N.join_forward(t["residual"], t["branch"], *args)
    want = (h, y, *N.join_backward(h, y, h, t["branch"], *args))
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(s):
            h2, y2 = N.join_forward(t["residual"], t["branch"], *args)
            got = (h2, y2, *N.join_backward(h2, y2, h2, t["branch"], *args))
        N.join_forward(t["residual"], t["branch"], *args)
        s.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_refusals(N):
    x, w = torch.ones(4, 6, 16, device="cuda"), torch.ones(16, device="cuda")
    b = x.bfloat16()
    for error, call in [
            (TypeError, lambda: N.norm_forward(x.half(), w)), (TypeError, lambda: N.norm_forward(x.cpu(), w)),
            (TypeError, lambda: N.norm_forward(x, w.half())), (ValueError, lambda: N.norm_forward(x, w[:15])),
            (ValueError, lambda: N.norm_forward(x, x)), (ValueError, lambda: N.norm_forward(x[0, 0, 0], w)),
            (ValueError, lambda: N.norm_forward(x, w, eps=0.0)), (ValueError, lambda: N.norm_forward(x, w, eps=-1.0)),
            (ValueError, lambda: N.norm_forward(torch.ones(2, 16392, device="cuda"), torch.ones(16392, device="cuda"))),
            (TypeError, lambda: N.norm_backward(b, x, w)), (ValueError, lambda: N.norm_backward(x[:3], x, w)),
            (TypeError, lambda: N.join_forward(b, x)), (ValueError, lambda: N.join_forward(x, x[:3])),
            (ValueError, lambda: N.join_forward(x, x, scale=float("nan"))),
            (ValueError, lambda: N.join_forward(x, x, gate=torch.ones(6, 16, device="cuda"))),
            (ValueError, lambda: N.join_forward(x, x, gate=torch.ones(4, 1, 1, device="cuda"))),
            (ValueError, lambda: N.join_forward(x, x, gate=torch.ones(1, 6, 16, device="cuda"))),
            (ValueError, lambda: N.join_forward(x, x, gate=torch.ones(1, 4, 6, 16, device="cuda"))),
            (ValueError, lambda: N.join_backward(x, x, x, x)), (TypeError, lambda: N.join_backward(b, x, x, x, w)),
            (TypeError, lambda: N.join_backward(x, x, x, b, w)), (ValueError, lambda: N.join_backward(x[:1], x, x, x, w))]:
        with pytest.raises(error):
            call()
