"""Rows further apart than a join reads them, without a GPU (memory that is never touched is never there)."""

import pytest
import torch


@pytest.fixture
def N(monkeypatch):
    from lookatmyquant_b200 import norms
    monkeypatch.setattr(norms, "_code", lambda x, what: 0)  # tensors of the host stand in
    return norms


@pytest.mark.parametrize("stride,kept", [(2**29 - 1, True), (2**29, False), (2**30 + 3, False)])
def test_rows_far_apart(N, stride, kept):
    """The last tokens of long texts: what the library takes a join's rows at (below 2^29 elements) is read in place, others go
    through a copy; the norm alone reads either."""
    base = torch.empty(stride + 8, dtype=torch.bfloat16)
    x = torch.as_strided(base, (2, 8), (stride, 1))
    x.copy_(torch.arange(16.0).view(2, 8))
    y, rows = N._rows(x)
    assert torch.equal(x, y) and (y is x) == kept and rows == (y.data_ptr(), 1 << 30, stride if kept else 8, 0)
    assert N._rows(x, 2) == (x, (x.data_ptr(), 1 << 30, stride, 0))
