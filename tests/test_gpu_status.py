"""The status words of the training operators: what check_status() sees, and calls inside CUDA graphs."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_check_status_waits_for_every_stream():
    """A bad id of a lookup that another stream has yet to run is reported, and reported once."""
    from lookatmyquant_b200 import embedding as E
    t = torch.randn(10, 16, device="cuda")
    bad = torch.tensor([1, 99], device="cuda")
    E.lookup(t, bad % 10)
    E.check_status()
    s = torch.cuda.Stream()
    for _ in range(3):
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            torch.cuda._sleep(200_000_000)  # some 0.1 s
            E.lookup(t, bad)
        with pytest.raises(ValueError, match="outside the table"):
            E.check_status()
        assert s.query()
        E.check_status()


def test_a_first_call_in_a_graph_is_refused():
    from lookatmyquant_b200 import _lib
    words, x = _lib.StatusWord("x"), torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        with pytest.raises(_lib.LamqError, match="captured"):
            words.on(x.device)
        x += 1
    graph.replay()
    assert words.on(x.device).item() == 0 and x.tolist() == [1.0] * 4


OPERATORS = {
    "attention forward": ((2, 300, 4, 64), lambda A, E, N, x, ids: A.forward(x, x[:, :2], x[:, 2:])),
    "attention forward by keys": ((1, 2000, 2, 128), lambda A, E, N, x, ids: A.forward(x[:, :, :3], x, x)),
    "attention backward": ((2, 300, 4, 64), lambda A, E, N, x, ids: A.backward(
        x, x, x[:, :2], x[:, 2:], *A.forward(x, x[:, :2], x[:, 2:]))),
    "lookup": ((1, 1, 100, 64), lambda A, E, N, x, ids: (E.lookup(x[0, :, 0], ids % 100, 3.0),)),
    "gradient of few tokens": ((1, 1, 500, 64), lambda A, E, N, x, ids: (E.lookup_gradient(x[0, :, 0], ids[:500], 3000),)),
    "gradient of many tokens": ((1, 1, 3000, 64), lambda A, E, N, x, ids: (E.lookup_gradient(x[0, :, 0], ids, 3000),)),
    "newton-schulz": ((1, 200, 1, 300), lambda A, E, N, x, ids: (N.newton_schulz(x[0, 0]),)),
    "newton-schulz on pairs": ((1, 2305, 1, 2049), lambda A, E, N, x, ids: (N.newton_schulz(x[0, 0]),)),
}


@pytest.mark.parametrize("name", OPERATORS)
def test_graphs_hold_the_operators(name):
    """A captured call, replayed on new inputs, gives what a call gives, bit for bit."""
    from lookatmyquant_b200 import attention as A, embedding as E, orthogonal as N
    shape, call = OPERATORS[name]
    g = torch.Generator("cuda").manual_seed(4)
    x = torch.randn(*shape, device="cuda", generator=g).bfloat16().transpose(1, 2)
    ids = torch.randint(0, 3000, (3000,), device="cuda", generator=g)
    call(A, E, N, x, ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(A, E, N, x, ids)
    for _ in range(3):
        x.copy_(torch.randn(*x.shape, device="cuda", generator=g))
        ids.random_(0, 3000, generator=g)
        graph.replay()
        for a, b in zip(got, call(A, E, N, x, ids)):
            assert torch.equal(a, b)
    for m in (A, E, N):
        m.check_status()
