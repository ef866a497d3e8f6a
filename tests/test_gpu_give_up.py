"""Bounded device waits that run out: the call ends with a status, and what depended on the wait is left alone."""

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
HERE = Path(__file__).resolve().parent


def library(folder, name, *sources, flags=()):
    from lookatmyquant_b200 import build
    out = folder / f"{name}.so"
    objects = [folder / f"{name}_{Path(src).stem}.o" for src in (*sources, build.CSRC / "api.cu")]
    jobs = [subprocess.Popen([build.nvcc(), *build.ARCH, *build.NVCC_FLAGS, *flags, "-c", str(src), "-o", str(o)],
                             stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
            for src, o in zip((*sources, build.CSRC / "api.cu"), objects)]
    assert all(j.wait() == 0 for j in jobs)
    subprocess.run([build.nvcc(), *build.ARCH, "-shared", *map(str, objects), "-o", str(out)], check=True)
    return ctypes.CDLL(str(out))


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    return library(tmp_path_factory.mktemp("give_up"), "embed_give_up", HERE / "embed_give_up.cu")


@pytest.fixture(scope="module")
def hasty(tmp_path_factory):
    """The attention and Newton-Schulz kernels with waits that give up at their first look at the time. (What waits for
    copies to land before a CTA leaves keeps its limit.)"""
    from lookatmyquant_b200 import _lib, build
    lib = library(tmp_path_factory.mktemp("hasty"), "hasty", build.CSRC / "attention.cu", build.CSRC / "orthogonal.cu",
                  flags=("-DLAMQ_GIVE_UP_NS=0ull", "-DLAMQ_GIVE_UP_POLLS=1u"))
    for name, (res, args) in _lib.SIGNATURES.items():
        if name.startswith(("lamq_attention", "lamq_newton_schulz")):
            f = getattr(lib, name)
            f.restype, f.argtypes = res, args
    return lib


@pytest.mark.parametrize("before_status", [0, 1])
def test_a_sort_that_gives_up_leaves_the_gradient_alone(harness, before_status):
    """The kernels after the sort do not go by keys and positions that nobody wrote: the gradient that was to be added to
    stays as it was. (Here they hold valid places, so that a kernel that did go by them would be seen in the result.) The
    status says so, also where a bad id was met before."""
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


def newton_schulz_call(lib, G, out, ws, status):
    from lookatmyquant_b200 import _lib, orthogonal as N
    m, n = G.shape
    assert lib.lamq_newton_schulz(G.data_ptr(), 0, n, 0, 1, m, n, 5, N._coefficients(N.COEFFICIENTS, 5), 1e-7, out.data_ptr(),
                                  ws.data_ptr(), ws.numel(), status.data_ptr(), _lib.stream_ptr()) == _lib.LAMQ_OK


@pytest.mark.parametrize("m,n", [(2560, 2561), (2561, 2500), (300, 500)])
def test_newton_schulz_ends_when_its_waits_give_up(hasty, m, n):
    """CTAs give up between the products, each somewhere else; the calls end with the status. The same buffers then serve a
    call of the usual limits, whose result is right whatever the status word held before."""
    from lookatmyquant_b200 import _lib, orthogonal as N
    lib = _lib.load()
    G = torch.randn(m, n, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    want = N.newton_schulz(G)
    ws = torch.empty(lib.lamq_newton_schulz_workspace_size(1, m, n), dtype=torch.uint8, device="cuda")
    out, status = torch.empty_like(want), torch.zeros(1, dtype=torch.int32, device="cuda")
    for _ in range(3):
        status.zero_()
        newton_schulz_call(hasty, G, out, ws, status)
        torch.cuda.synchronize()
        assert status.item() == 4
    for _ in range(3):
        out.zero_()
        newton_schulz_call(lib, G, out, ws, status)
        assert torch.equal(out, want) and status.item() == 4
    N.check_status()


@pytest.mark.parametrize("Lq,Lk,D", [(900, 900, 64), (900, 900, 128), (5, 2000, 128)])
def test_attention_ends_when_its_waits_give_up(hasty, Lq, Lk, D):
    from lookatmyquant_b200 import _lib, attention as A
    g = torch.Generator("cuda").manual_seed(3)
    rand = lambda H, L: torch.randn(2, L, H, D, device="cuda", generator=g).bfloat16().transpose(1, 2)
    q, k, v, do = rand(8, Lq), rand(2, Lk), rand(2, Lk), rand(8, Lq)
    o, lse = A.forward(q, k, v)
    want = (o, lse, *A.backward(do, q, k, v, o, lse))
    got = [x.clone() for x in want]
    size = _lib.load().lamq_attention_backward_workspace_size(2, 8, Lq)
    ws, status = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    heads = lambda x: (x.data_ptr(), *x.stride()[:3])
    args = _lib.ATTENTION_ARGS.pack(2, 8, 2, D, True, Lq, Lk, D**-0.5, 0, 0, 0, *heads(q), *heads(k), *heads(v), *heads(got[0]),
                                    got[1].data_ptr(), *heads(do), *(y for x in got[2:] for y in heads(x)))
    calls = {"forward": lambda lib: lib.lamq_attention_forward(args, status.data_ptr(), _lib.stream_ptr()),
             "backward": lambda lib: lib.lamq_attention_backward(args, ws.data_ptr(), size, status.data_ptr(),
                                                                 _lib.stream_ptr())}
    for call in calls.values():
        for _ in range(3):
            status.zero_()
            assert call(hasty) == _lib.LAMQ_OK
            torch.cuda.synchronize()
            assert status.item() == 4
    for _ in range(3):
        for x in got:
            x.zero_()
        assert calls["forward"](_lib.load()) == calls["backward"](_lib.load()) == _lib.LAMQ_OK
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    A.check_status()


def test_an_old_error_ends_no_later_call():
    """A status word that nobody has checked yet: the calls after it wait as long as ever."""
    from lookatmyquant_b200 import _lib, attention as A, orthogonal as N
    g = torch.Generator("cuda").manual_seed(5)
    x = torch.randn(2, 700, 8, 128, device="cuda", generator=g).bfloat16().transpose(1, 2)
    Gs = [torch.randn(*s, device="cuda", generator=g) for s in ((300, 500), (2560, 2561))]
    run = lambda: (*A.forward(x, x, x), *A.backward(x, x, x, x, *A.forward(x, x, x)), *(N.newton_schulz(G) for G in Gs))
    want = run()
    for m in (A, N):
        m._STATUS.on(x.device).fill_(4)
    torch.cuda.synchronize()
    for _ in range(5):
        for a, b in zip(run(), want):
            assert torch.equal(a, b)
    for m in (A, N):
        with pytest.raises(_lib.LamqError):
            m.check_status()
        m.check_status()
