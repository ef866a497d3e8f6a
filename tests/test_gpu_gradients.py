"""The global norm of many gradients and their clipping, against 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def G():
    from lookatmyquant_b200 import gradients
    return gradients


def exact_norm(tensors):
    return math.sqrt(sum(float(x.double().square().sum()) for x in tensors))


# fp32 sums of eight squares (seven roundings deep at most, each at most half a step of the sum; half of that in the root) and the
# fp32 result
NORM = 8 / 2 * 2.0**-24 + 2.0**-24


def make(shapes, dtype, seed=0, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return [(scale * (1 + i % 3) * torch.randn(s, device="cuda", generator=g)).to(dtype if dtype else (BF, FP)[i % 2])
            for i, s in enumerate(shapes)]


LISTS = {
    "one element": [(1,)], "a vector": [(7,)], "a tile": [(16384,)], "a tile and one": [(16385,), (8193,)],
    "a model": [(960, 960), (320, 960), (960,), (2560, 960), (5000, 960), (960,)],
    "odd": [(3,), (1337, 17), (0,), (129,), (33, 1000), ()],
    "many": [(17 + i % 400,) for i in range(300)], "more than a launch takes": [(1 + i % 77, 3) for i in range(2345)],
    "large": [(40_000_001,), (5,)],
}


@pytest.mark.parametrize("dtype", [BF, FP, None])
@pytest.mark.parametrize("name", LISTS)
def test_global_norm_and_clip(G, name, dtype):
    xs = make(LISTS[name], dtype)
    want = exact_norm(xs)
    norm = G.global_norm(xs)
    assert norm.shape == () and norm.dtype == FP
    assert abs(float(norm) - want) <= NORM * want
    bound = want / 3
    factor = bound / (want + 1e-6)
    for out_dtype in (None, BF, FP):
        ins = [x.clone() for x in xs]
        out = None if out_dtype is None else [torch.full_like(x, float("nan"), dtype=out_dtype) for x in ins]
        got = G.clip(ins, bound, out)
        assert torch.equal(got, norm)
        for x, y, z in zip(xs, ins if out is None else out, ins):
            # the factor from a norm off by NORM and rounded, the product rounded to fp32 and to its type
            exact = x.double() * factor
            allowed = exact.abs() * (NORM + 3 * 2.0**-24 + torch.finfo(y.dtype).eps / 2) + 1e-44
            assert bool(((y.double() - exact).abs() <= allowed).all())
            assert out is None or torch.equal(z, x)


def test_a_norm_within_the_bound_changes_nothing(G):
    xs = make(LISTS["a model"], None)
    norm = exact_norm(xs)
    kept = [x.clone() for x in xs]
    for bound in (norm * 1.001 + 2e-6, math.inf):
        G.clip(xs, bound)
        assert all(torch.equal(a, b) for a, b in zip(xs, kept))
        out = [torch.zeros_like(x) for x in xs]
        G.clip(xs, bound, out)
        assert all(torch.equal(a, b) for a, b in zip(out, kept))
    G.clip(xs, 0.0)
    assert all(float(x.abs().sum()) == 0 for x in xs)


@pytest.mark.parametrize("scale", [1e-44, 1e-30, 1e-22, 1e-19, 1e15, 1e19, 1e25, 3e37])
@pytest.mark.parametrize("n", [1, 8, 100, 100_003])
def test_norms_at_the_ends_of_fp32(G, scale, n):
    """Squares that fp32 would lose or overflow, beside ones that it holds."""
    xs = make([(n,), (n,)], FP, 3, scale)
    want = exact_norm(xs)
    if want < 3.4e38:
        assert abs(float(G.global_norm(xs)) - want) <= NORM * want + 1e-45
    else:
        assert float(G.global_norm(xs)) == math.inf
    ys = [x.clone() for x in xs]
    G.clip(ys, 1e-3 * want)
    for x, y in zip(xs, ys):
        exact = x.double() * (1e-3 * want / (want + 1e-6))
        assert bool(((y.double() - exact).abs() <= exact.abs() * (NORM + 4 * 2.0**-24) + 1.5e-45).all())
    mixed = xs + make([(n,)], FP, 4, 1.0)
    want = exact_norm(mixed)
    assert abs(float(G.global_norm(mixed)) - want) <= NORM * want or want > 3.4e38


def test_clipping_of_a_vast_norm(G):
    """A factor below fp32's range does not flush the values that it takes."""
    xs = [torch.full((1000,), 3e38, device="cuda")]
    want = exact_norm(xs)
    G.clip(xs, 1e-5)
    exact = 3e38 * 1e-5 / want
    assert bool(((xs[0].double() / exact - 1).abs() <= NORM + 1e-6).all())


@pytest.mark.parametrize("where", [0, 5, 16384, 40_000])
def test_what_is_not_finite(G, where):
    for bad in (math.nan, math.inf, -math.inf):
        for dtype in (BF, FP):
            xs = make([(3, 7), (50_001,)], dtype)
            xs[1][where] = bad
            norm = float(G.global_norm(xs))
            assert math.isnan(norm) if math.isnan(bad) else norm == math.inf
            G.clip(xs, 1.0)
            if math.isnan(bad):
                assert all(bool(x.isnan().all()) for x in xs)
            else:
                assert bool(xs[1][where].isnan()) and float(xs[0].abs().sum()) == 0
                xs[1][where] = 0
                assert float(xs[1].abs().sum()) == 0


def test_zeros(G):
    xs = [torch.zeros(1000, 33, device="cuda"), torch.zeros(5, device="cuda").bfloat16()]
    assert float(G.global_norm(xs)) == 0
    G.clip(xs, 1.0)
    assert float(xs[0].abs().sum()) == 0
    assert float(G.global_norm([torch.zeros(0, device="cuda")])) == 0
    assert float(G.clip([torch.zeros(0, device="cuda"), None], 1.0)) == 0


def test_tensors_that_lie_anywhere(G):
    """Other orders of the axes, slices, tensors that start between two 16-byte pieces, None; outputs of other strides."""
    base = make([(200, 300)], FP)[0]
    flat = make([(5001,)], BF, 1)[0]

    def views(b, f):
        return [b.t(), None, b[:0], f[1:4000], f[4001:]]

    def sliced(b):
        return [b[:, ::2], b[:, 1::2]]
    for pick in (lambda b, f: views(b, f), lambda b, f: sliced(b) + [f[3:]]):
        b, f = base.clone(), flat.clone()
        xs = pick(b, f)
        plain = [x.clone(memory_format=torch.contiguous_format) for x in xs if x is not None]
        want = exact_norm(plain)
        assert abs(float(G.global_norm(xs)) - want) <= NORM * want
        out = [None if x is None else torch.zeros(x.shape, device="cuda") for x in xs]
        out[0] = torch.zeros(xs[0].shape[::-1], device="cuda").t()
        G.clip(xs, want / 2, out)
        into = [None if x is None else torch.zeros(2 * x.numel(), device="cuda")[::2].view(x.shape) for x in xs]
        G.clip(xs, want / 2, into)
        G.clip(xs, want / 2)
        G.clip(plain, want / 2)
        got = [x for x in xs if x is not None]
        for x, y, o, i in zip(got, plain, [o for o in out if o is not None], [i for i in into if i is not None]):
            assert torch.equal(x, y)
            assert torch.equal(o.to(x.dtype), x) and torch.equal(i, o)
    assert torch.equal(b[:, 0].isnan(), torch.zeros(200, dtype=torch.bool, device="cuda"))


def test_equal_calls_give_equal_bits_also_in_graphs(G):
    xs = make(LISTS["a model"] + LISTS["many"], None)
    first = G.global_norm(xs)
    assert all(torch.equal(first, G.global_norm(xs)) for _ in range(5))
    out = [torch.empty_like(x) for x in xs]
    G.clip(xs, 1.0, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = G.clip(xs, 1.0, out)
    for k in range(3):
        for x, y in zip(xs, make(LISTS["a model"] + LISTS["many"], None, 10 + k)):
            x.copy_(y)
        graph.replay()
        ys = [x.clone() for x in xs]
        assert torch.equal(norm, G.clip(ys, 1.0))
        assert all(torch.equal(a, b) for a, b in zip(out, ys))


def test_two_streams_at_once(G):
    lists = [make(LISTS["a model"], FP, s) for s in (1, 2)]
    want = [G.global_norm(xs) for xs in lists]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for xs, s in zip(lists, streams):
            with torch.cuda.stream(s):
                got.append(G.global_norm(xs))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_clipping_is_a_change_that_autograd_sees(G):
    x = torch.ones(8, device="cuda").requires_grad_(True)
    y = x * 2
    z = y.square().sum()
    with torch.no_grad():
        G.clip([y], 0.5)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_clipping_in_inference_mode(G):
    with torch.inference_mode():
        x = torch.full((100,), 2.0, device="cuda")
        assert abs(float(G.clip([x], 10.0)) - 20.0) <= 1e-4 and bool(((x - 1.0).abs() <= 1e-6).all())


def test_refusals(G):
    x = torch.ones(8, 8, device="cuda")
    for error, call in [
            (ValueError, lambda: G.global_norm([])), (ValueError, lambda: G.global_norm([None])),
            (TypeError, lambda: G.global_norm([x.half()])), (TypeError, lambda: G.global_norm([x.cpu()])),
            (TypeError, lambda: G.global_norm([x.to_sparse()])), (TypeError, lambda: G.global_norm([1.0])),
            (ValueError, lambda: G.clip([x], -1.0)), (ValueError, lambda: G.clip([x], math.nan)),
            (ValueError, lambda: G.clip([x], 1.0, eps=-1.0)), (ValueError, lambda: G.clip([x, x], 1.0)),
            (ValueError, lambda: G.clip([x, x[4:]], 1.0)), (ValueError, lambda: G.clip([x[:, ::2], x[:, ::2]], 1.0)), (ValueError, lambda: G.clip([x], 1.0, [x.flatten()])),
            (ValueError, lambda: G.clip([x], 1.0, [])), (ValueError, lambda: G.clip([x[:4]], 1.0, [x[2:6]])),
            (TypeError, lambda: G.clip([x], 1.0, [x.half()])), (TypeError, lambda: G.clip([x], 1.0, [None]))]:
        with pytest.raises(error):
            call()
    assert bool((x == 1).all())
