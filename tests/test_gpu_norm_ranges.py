"""The norms' gradients where the products of a gradient and a row leave fp32's range, though the row's squares, the normed row
and the result are within it: the mean of t · ĥ is then that of the normed row."""

import pytest
import torch
from step_reference import assert_close, join_backward, norm_gradient
from test_gpu_norms import BF, FP, N, generator, values  # noqa: F401  (N: the module under test)

pytestmark = pytest.mark.gpu

WIDTHS = [8, 24, 33, 128, 960, 1337, 4096, 4104, 8200, 9728, 16383, 16384]
# the sizes of h and of dy, and eps: products past 3e38 (sums of 16384 of them, too); products below fp32's smallest numbers
ENDS = [(1e16, 1e23, 1e-6), (1e18, 1e20, 1e-6), (1e-13, 1e-31, 1e-30), (1e-17, 1e-33, 1e-36)]


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("h,dy,eps", ENDS, ids=["large", "large rows", "small", "smallest"])
def test_norm_backward(N, d, dtype, h, dy, eps):  # noqa: F811
    """Every other row at such an end, beside ordinary ones, whose results are the same bits as without them."""
    g = generator(d)
    n = 37
    x, w, grad = values(g, n, d), values(g, d, dtype=dtype), values(g, n, d, scale=1e-3)
    plain = [t.to(dtype) for t in (x, grad)]
    x[::2] *= h
    grad[::2] *= 1e3 * dy
    x, grad = x.to(dtype), grad.to(dtype)
    dx, dw = N.norm_backward(grad, x, w, eps=eps)
    wx, ww = norm_gradient(grad.double(), torch.zeros_like(x).double(), x.double(), w, eps, 0.0)
    assert_close(dx, wx, "dx")
    assert_close(dw, ww, "dw")
    assert torch.equal(dx[1::2], N.norm_backward(plain[1], plain[0], w, eps=eps)[0][1::2])


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("h,dy,eps", ENDS[:3], ids=["large", "large rows", "small"])
def test_join_backward(N, d, h, dy, eps):  # noqa: F811
    g = generator(d + 1)
    shape = (3, 11, d)
    stream, branch = values(g, *shape, scale=h), values(g, *shape)
    w, post, gate = values(g, d), values(g, d), values(g, 3, 1, d)
    dh, grad = values(g, *shape, scale=dy / h), values(g, *shape, scale=dy)
    for rest in ((w, post, gate), (w, None, None)):
        got = dict(zip(("residual", "branch", "weight", "post", "gate"), N.join_backward(dh, grad, stream, branch, *rest, 0.5, eps)))
        for k, x in join_backward(dh, grad, stream, branch, *rest, 0.5, eps).items():
            assert_close(got[k], x, f"d_{k}")
