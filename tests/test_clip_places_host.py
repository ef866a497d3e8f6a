"""Where clipped values go, without a GPU: a stand-in for the library reads and writes the memory that the call describes, and
refuses, as the library does, outputs that meet one another or another tensor's input."""

import ctypes

import pytest
import torch


def at(pointer, n):
    return torch.frombuffer((ctypes.c_float * n).from_address(pointer), dtype=torch.float32) if n else torch.zeros(0)


@pytest.fixture
def G(monkeypatch):
    from lookatmyquant_b200 import gradients

    def call(name, values, count, device, max_norm, eps):
        rows = [values[5 * i:5 * i + 5] for i in range(count)]
        writes = [(out, out + 4 * n, i) for i, (_, out, n, _, _) in enumerate(rows)]
        reads = [(p, p + 4 * n, i if p == out else -1) for i, (p, out, n, _, _) in enumerate(rows)]
        if any(a < d and c < b and i != j for a, b, i in writes for c, d, j in writes + reads):
            raise ValueError("overlap")
        norm = sum(at(p, n).double().square().sum() for p, _, n, _, _ in rows).sqrt()
        scaled = [at(p, n) * min(1.0, max_norm / (float(norm) + eps)) for p, _, n, _, _ in rows]
        for (_, out, n, _, _), x in zip(rows, scaled):
            at(out, n).copy_(x)
        return norm.float()
    monkeypatch.setattr(gradients, "_code", lambda *_: 0)
    monkeypatch.setattr(gradients, "_call", call)
    return gradients


def test_two_outputs_in_one_view_with_gaps_are_refused(G):
    xs = [torch.ones(4, 3), torch.full((4, 3), 2.0)]
    base = torch.zeros(4, 6)
    for out in ([base[:, :3], base[:, :3]], [base[:, ::2], base[:, ::2]]):
        with pytest.raises(ValueError, match="overlap"):
            G.clip(xs, 1.0, out)
        assert float(base.abs().sum()) == 0
    with pytest.raises(ValueError, match="overlap"):  # in place and an output
        G.clip([base[:, :3], xs[0]], 1.0, [base[:, :3], base[:, :3]])
    G.clip(xs, 1.0, [base[:, :3], base[:, 3:]])
    norm = 60.0**0.5
    assert torch.allclose(base, torch.cat(xs, 1) / norm, rtol=1e-5)


def test_outputs_in_another_order_of_the_axes_are_seen_where_they_lie(G):
    xs = [torch.ones(4, 3), torch.full((3, 4), 2.0)]
    out = torch.zeros(3, 4)
    with pytest.raises(ValueError, match="overlap"):
        G.clip(xs, 1.0, [out.t(), out])
    assert float(out.abs().sum()) == 0
    G.clip(xs, 1.0, [out.t(), torch.zeros(3, 4)])
    assert torch.allclose(out, torch.full((3, 4), 60**-0.5), rtol=1e-5)


def test_tensors_that_overlap_themselves_are_refused_before_anything_changes(G):
    x, wide = torch.full((8,), 3.0), torch.ones(3, 1).expand(3, 4)
    for call in (lambda: G.clip([x, wide], 1.0), lambda: G.clip([x, torch.ones(3, 4)], 1.0, [x, wide]),
                 lambda: G.clip([x, torch.ones(2, 3)], 1.0, [x, torch.zeros(3).expand(2, 3)])):
        with pytest.raises(ValueError, match="overlap"):
            call()
        assert bool((x == 3).all()) and bool((wide == 1).all())
    G.clip([x, torch.ones(3, 1).expand(3, 1)], 1.0)  # one entry along the axis
    out = torch.zeros(3, 4)
    G.clip([wide], 1.0, [out])  # read only
    assert torch.allclose(out, torch.full((3, 4), 12**-0.5), rtol=1e-5)


def test_views_of_inference_mode_are_written_outside_it(G):
    with torch.inference_mode():
        base = torch.full((4, 6), 2.0)
        view = base[:, :3]
    x = torch.full((5,), 1.0)
    G.clip([x, view], 1.0)
    norm = 53.0**0.5
    assert torch.allclose(view, torch.full((4, 3), 2 / norm), rtol=1e-5) and bool((base[:, 3:] == 2).all())
    assert torch.allclose(x, torch.full((5,), 1 / norm), rtol=1e-5)
