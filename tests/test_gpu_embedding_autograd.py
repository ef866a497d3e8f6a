"""scaled_embedding under autograd against torch's embedding."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("padding", [None, 0, 7, 39, -1, -40])
def test_padding_is_torchs(padding):
    """A table whose padding row is not zero: the row is looked up as it is stored, and gets no gradient. Powers of two as
    scale and small integers as values: every sum is exact."""
    from lookatmyquant_b200 import embedding as E
    g = torch.Generator("cuda").manual_seed(1)
    t = torch.randint(-8, 9, (40, 24), device="cuda", generator=g).float()
    ids = torch.randint(0, 40, (3, 50), device="cuda", generator=g)
    ids[0, :5] = 0 if padding is None else padding % 40
    c = torch.randint(-8, 9, (3, 50, 24), device="cuda", generator=g).float()
    mine, want = t.clone().requires_grad_(True), t.clone().requires_grad_(True)
    y = E.scaled_embedding(mine, ids, 4.0, padding)
    w = torch.nn.functional.embedding(ids, want, padding_idx=padding) * 4.0
    assert torch.equal(y, w)
    (y * c).sum().backward()
    (w * c).sum().backward()
    assert torch.equal(mine.grad, want.grad)
    with pytest.raises(ValueError):
        E.scaled_embedding(mine, ids, 4.0, 40)
    with pytest.raises(ValueError):
        E.scaled_embedding(mine, ids, 4.0, -41)
    E.check_status()


@pytest.mark.parametrize("padding", [None, 3])
def test_second_derivatives_are_torchs(padding):
    """A penalty on the first gradients, differentiated again (and a third time through the lookup of the second), against
    torch's embedding in 64 bits: every value passes a dozen fp32 operations on numbers of like magnitude."""
    from lookatmyquant_b200 import embedding as E
    g = torch.Generator("cuda").manual_seed(2)
    t = torch.randn(12, 8, device="cuda", generator=g)
    ids = torch.randint(0, 12, (40,), device="cuda", generator=g)
    got = {}
    for name, table in (("mine", t.clone()), ("torch", t.double())):
        table.requires_grad_(True)
        look = (lambda: E.scaled_embedding(table, ids, 0.5, padding)) if name == "mine" else (
            lambda: torch.nn.functional.embedding(ids, table, padding_idx=padding) * 0.5)
        first, = torch.autograd.grad(look().pow(4).sum(), table, create_graph=True)
        second, = torch.autograd.grad(first.square().sum() + look().square().sum(), table, create_graph=True)
        third, = torch.autograd.grad(second.square().sum(), table)
        got[name] = first, second, third
    for a, b in zip(got["mine"], got["torch"]):
        assert float((a.detach().double() - b.detach()).norm()) <= 1e-4 * float(b.detach().norm())
        assert padding is None or float(a[padding].abs().sum()) == 0
