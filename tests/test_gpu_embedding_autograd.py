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
