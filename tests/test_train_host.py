"""The training operators' host side without a GPU: stand-ins take the kernels' place."""

import contextlib
import threading
import time

import pytest
import torch


def test_threads_share_one_status_word(monkeypatch):
    """Whichever threads make a device's first call: they get the word that check() reads."""
    from lookatmyquant_b200 import _lib
    zeros = torch.zeros

    def slow_zeros(*a, device=None, **kw):
        time.sleep(0.05)
        return zeros(*a, **kw)
    monkeypatch.setattr(torch, "zeros", slow_zeros)
    monkeypatch.setattr(torch.cuda, "device", contextlib.nullcontext)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    words, got = _lib.StatusWord("x"), []
    threads = [threading.Thread(target=lambda: got.append(words.on(torch.device("cuda", 0)))) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 4 and all(w is words.on(torch.device("cuda", 0)) for w in got)


def test_each_error_has_its_own_words(monkeypatch):
    from lookatmyquant_b200 import _lib, embedding, orthogonal
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    for words, code, error, text in ((embedding._STATUS, _lib.LAMQ_ERR_INVALID, ValueError, "outside the table"),
                                     (embedding._STATUS, _lib.LAMQ_ERR_TIMEOUT, _lib.LamqError, "gave up on a device wait"),
                                     (orthogonal._STATUS, _lib.LAMQ_ERR_TIMEOUT, _lib.LamqError, "newton_schulz.*gave up")):
        monkeypatch.setattr(words, "words", {torch.device("cuda", 0): torch.tensor([code], dtype=torch.int32)})
        with pytest.raises(error, match=text) as e:
            words.check()
        assert code != _lib.LAMQ_ERR_TIMEOUT or "outside" not in str(e.value)
        words.check()


def test_negative_padding_indices_count_from_the_end():
    from lookatmyquant_b200 import embedding
    assert [embedding._padding(p, 40) for p in (None, 0, 39, -1, -40)] == [-1, 0, 39, 39, 0]
    for p, rows in ((40, 40), (-41, 40), (0, 0), (-1, 0)):
        with pytest.raises(ValueError):
            embedding._padding(p, rows)


def stand_ins_for_attention(monkeypatch):
    from lookatmyquant_b200 import attention as A
    monkeypatch.setattr(A, "forward", lambda q, k, v, *a: (q * k * v, q.detach().sum(-1)))
    monkeypatch.setattr(A, "backward", lambda do, q, k, v, *a: (do * k * v, do * q * v, do * q * k))
    return A


def test_second_derivatives_of_attention_raise(monkeypatch):
    """Gradients come from kernels that autograd does not see; what is differentiated through them must not take them for
    constants."""
    A = stand_ins_for_attention(monkeypatch)
    q, k, v = (torch.randn(1, 2, 3, 8).requires_grad_(True) for _ in range(3))
    first = torch.autograd.grad(A.attention(q, k, v).sum(), (q, k, v), create_graph=True)
    assert torch.equal(first[0], k * v)
    with pytest.raises(RuntimeError, match="no second derivatives"):
        torch.autograd.grad(first[0].square().sum() + q.sum(), q)
    c = torch.randn(1, 2, 3, 8).requires_grad_(True)
    first = torch.autograd.grad((A.attention(q, k, v) * c).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivatives"):
        torch.autograd.grad(first[0].sum(), c)
    A.attention(q, k, v).sum().backward()  # a first derivative alone is none of its business
    assert torch.equal(q.grad, k * v) and not q.grad.requires_grad


def muon_run(monkeypatch, dtype, reload):
    """Six Muon steps on two matrices, through a state dict after three of them: parameters and momenta."""
    from lookatmyquant_b200 import orthogonal as N
    monkeypatch.setattr(N, "newton_schulz", lambda G, steps, coefficients: (G / G.norm()).bfloat16())
    g = torch.Generator().manual_seed(1)
    params = [torch.nn.Parameter(torch.randn(*s, generator=g).to(dtype)) for s in ((8, 5), (3, 7))]
    opt = N.Muon(params, lr=0.1, weight_decay=0.01)
    for step in range(6):
        if step == 3 and reload:
            state = opt.state_dict()
            params = [torch.nn.Parameter(p.detach().clone()) for p in params]
            opt = N.Muon(params, lr=0.5)
            opt.load_state_dict(state)
        for p in params:
            p.grad = torch.randn(p.shape, generator=g).to(dtype)
        opt.step()
    return [p.detach() for p in params] + [opt.state[p]["momentum"] for p in params]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_muon_goes_on_from_a_state_dict_as_if_nothing_had_been(monkeypatch, dtype):
    want, got = muon_run(monkeypatch, dtype, False), muon_run(monkeypatch, dtype, True)
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a, b)
    assert got[2].dtype == got[3].dtype == torch.float32


def test_muon_shares_no_buffer_with_the_state_dict_it_loaded(monkeypatch):
    from lookatmyquant_b200 import orthogonal as N
    monkeypatch.setattr(N, "newton_schulz", lambda G, steps, coefficients: G.bfloat16())
    p = torch.nn.Parameter(torch.ones(2, 2))
    first, second = N.Muon([p]), N.Muon([p])
    p.grad = torch.ones(2, 2)
    first.step()
    second.load_state_dict(first.state_dict())
    second.step()
    assert torch.equal(first.state[p]["momentum"], torch.ones(2, 2))
    assert torch.equal(second.state[p]["momentum"], torch.full((2, 2), 1.95))


def test_muon_makes_a_momentum_once(monkeypatch):
    from lookatmyquant_b200 import orthogonal as N
    monkeypatch.setattr(N, "newton_schulz", lambda G, steps, coefficients: G.bfloat16())
    made, zeros_like = [], torch.zeros_like
    monkeypatch.setattr(torch, "zeros_like", lambda *a, **kw: made.append(1) or zeros_like(*a, **kw))
    params = [torch.nn.Parameter(torch.ones(2, 3)) for _ in range(3)]
    opt = N.Muon(params)
    for _ in range(4):
        for p in params:
            p.grad = torch.ones(2, 3)
        opt.step()
    assert len(made) == 3


def test_muon_steps_over_empty_matrices(monkeypatch):
    from lookatmyquant_b200 import orthogonal as N
    monkeypatch.setattr(N, "newton_schulz", lambda G, steps, coefficients: G.bfloat16())
    params = [torch.nn.Parameter(torch.ones(*s)) for s in ((3, 0), (0, 3), (2, 2))]
    opt = N.Muon(params, lr=0.5, nesterov=False)
    for p in params:
        p.grad = torch.ones_like(p)
    opt.step()
    assert [p.shape for p in params] == [(3, 0), (0, 3), (2, 2)] and torch.equal(params[2], torch.full((2, 2), 0.5))
