"""Bounded device waits that run out: the call ends with a status, and what depended on the wait is left alone."""

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
HERE = Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    from lookatmyquant_b200 import build
    out = tmp_path_factory.mktemp("give_up") / "embed_give_up.so"
    subprocess.run([build.nvcc(), *build.ARCH, *build.NVCC_FLAGS, "-shared", str(HERE / "embed_give_up.cu"),
                    str(build.CSRC / "api.cu"), "-o", str(out)], check=True, capture_output=True)
    return ctypes.CDLL(str(out))


@pytest.mark.parametrize("before_status", [0, 1])
def test_a_sort_that_gives_up_leaves_the_gradient_alone(harness, before_status):
    """The kernels after the sort do not go by keys and positions that nobody wrote: the gradient that was to be added to
    stays as it was. (Here they hold valid places, so that a kernel that did go by them would be seen in the result.) The status says so, also where a bad id was met before."""
    n, rows, d = 3000, 100, 64
    g = torch.Generator("cuda").manual_seed(1)
    dy = torch.randn(n, d, device="cuda", generator=g)
    ids = torch.randint(0, rows, (n,), device="cuda", generator=g)
    dE = torch.randn(rows, d, device="cuda", generator=g)
    before = dE.clone()
    keys = (torch.arange(n, device="cuda", dtype=torch.int32) * rows // n).repeat(2)
    pos = torch.arange(n, device="cuda", dtype=torch.int32).repeat(2)
    counts = torch.zeros(64 * 512, dtype=torch.int32, device="cuda")
    head, tail = torch.zeros(n, d, device="cuda"), torch.zeros(n, d, device="cuda")
    words, status = (torch.zeros(2, dtype=torch.int32, device="cuda") for _ in range(2))
    status[0] = before_status
    torch.cuda.synchronize()
    p = lambda t: ctypes.c_void_p(t.data_ptr())
    err = harness.gradient_with_a_block_missing(p(dy), p(ids), ctypes.c_int64(n), ctypes.c_int64(rows), d, p(dE), p(keys),
                                                p(pos), p(counts), p(head), p(tail), p(words), p(status))
    assert err == 0
    assert status.tolist() == [4, 0] and words.tolist() == [1, 1]  # LAMQ_ERR_TIMEOUT; one arrival, given up
    assert torch.equal(dE, before)


@pytest.mark.parametrize("m,n", [(2560, 2561), (2561, 2500), (300, 500)])
def test_newton_schulz_ends_where_an_error_has_been_recorded(m, n):
    """Every CTA gives up at its next wait, somewhere between the products; the call ends, and the next one is right."""
    from lookatmyquant_b200 import _lib, orthogonal as N
    lib = _lib.load()
    G = torch.randn(m, n, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    want = N.newton_schulz(G)
    ws = torch.empty(lib.lamq_newton_schulz_workspace_size(1, m, n), dtype=torch.uint8, device="cuda")
    out, status = torch.empty_like(want), torch.full((1,), 4, dtype=torch.int32, device="cuda")
    call = lambda: lib.lamq_newton_schulz(G.data_ptr(), 0, n, 0, 1, m, n, 5, N._coefficients(N.COEFFICIENTS, 5), 1e-7,
                                          out.data_ptr(), ws.data_ptr(), ws.numel(), status.data_ptr(), _lib.stream_ptr())
    for _ in range(3):
        assert call() == _lib.LAMQ_OK
    torch.cuda.synchronize()
    assert status.item() == 4
    status.zero_()
    assert call() == _lib.LAMQ_OK
    assert torch.equal(out, want) and status.item() == 0
    N.check_status()


@pytest.mark.parametrize("Lq,Lk,D", [(900, 900, 64), (900, 900, 128), (5, 2000, 128)])
def test_attention_ends_where_an_error_has_been_recorded(Lq, Lk, D):
    """Threads that wait long enough to look give up, wherever they are; the calls end, and the next ones are right."""
    from lookatmyquant_b200 import _lib, attention as A
    lib = _lib.load()
    g = torch.Generator("cuda").manual_seed(3)
    rand = lambda H, L: torch.randn(2, L, H, D, device="cuda", generator=g).bfloat16().transpose(1, 2)
    q, k, v, do = rand(8, Lq), rand(2, Lk), rand(2, Lk), rand(8, Lq)
    o, lse = A.forward(q, k, v)
    want = (o, lse, *A.backward(do, q, k, v, o, lse))
    got = [torch.empty_like(x) for x in want]
    size = lib.lamq_attention_backward_workspace_size(2, 8, Lq)
    ws, status = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.full((1,), 4, dtype=torch.int32, device="cuda")
    heads = lambda x: (x.data_ptr(), *x.stride()[:3])
    args = _lib.ATTENTION_ARGS.pack(2, 8, 2, D, True, Lq, Lk, D**-0.5, 0, 0, 0, *heads(q), *heads(k), *heads(v), *heads(got[0]),
                                    got[1].data_ptr(), *heads(do), *(y for x in got[2:] for y in heads(x)))

    def calls():
        assert lib.lamq_attention_forward(args, status.data_ptr(), _lib.stream_ptr()) == _lib.LAMQ_OK
        assert lib.lamq_attention_backward(args, ws.data_ptr(), size, status.data_ptr(), _lib.stream_ptr()) == _lib.LAMQ_OK
    for _ in range(3):
        calls()
    torch.cuda.synchronize()
    assert status.item() == 4
    status.zero_()
    calls()
    assert status.item() == 0
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    A.check_status()
