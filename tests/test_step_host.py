"""The host side of the norms and of the gradients' norm without a GPU: rows, gates and memory as the calls describe them."""

import pytest
import torch


@pytest.fixture
def N(monkeypatch):
    from lookatmyquant_b200 import norms
    monkeypatch.setattr(norms, "_code", lambda x, what: 0)  # tensors of the host stand in
    return norms


def element(x, rows, i, j):
    """What the library reads as element j of row i."""
    _, inner, row, outer = rows
    flat = torch.as_strided(x, (x.untyped_storage().size() // 4 - x.storage_offset(),), (1,), x.storage_offset())
    return flat[(i // inner) * outer + (i % inner) * row + j]


@pytest.mark.parametrize("strides", [1, 2])
def test_rows_are_described_as_they_lie(N, strides):
    base = torch.arange(2 * 6 * 10 * 8.0).view(2, 6, 10, 8)
    views = [base, base[:, :, 2:5], base[:, ::2], base[1], base[0, 0, 0], base[:, :1], base[:, :, :1], base[..., 1:4], base[..., :1],
             base.transpose(1, 2), base[..., ::2], base[:1, 2:3, :, :], base[0, :, 3], base[:, 1, 4].expand(3, 2, 8), base[:, :, 3],
             base.permute(3, 0, 1, 2)]
    for x in views:
        y, rows = N._rows(x, strides)
        assert torch.equal(x, y) and rows[0] == y.data_ptr() and rows[1] >= 1
        if y is not x:
            assert y.is_contiguous()
        flat = x.reshape(-1, x.shape[-1])
        if strides == 1:
            assert rows[1] >= len(flat)
        for i in range(len(flat)):
            for j in (0, x.shape[-1] - 1):
                assert element(y, rows, i, j) == flat[i, j]


def test_gates_span_the_rows_that_share_them(N):
    b = torch.zeros(3, 4, 5, 8)
    for shape, span in (((8,), 60), ((1, 8), 60), ((1, 1, 1, 8), 60), ((3, 1, 1, 8), 20), ((3, 4, 1, 8), 5), ((3, 4, 5, 8), 1)):
        assert N._gate(torch.zeros(shape), b)[2] == span
    assert N._gate(torch.zeros(1, 4, 8), torch.zeros(1, 4, 8))[2] == 1 and N._gate(torch.zeros(1, 1, 8), torch.zeros(2, 1, 8))[2] == 2
    assert N._gate(torch.zeros(8).expand(3, 1, 1, 8), b)[0].is_contiguous()
    for shape in ((3, 4, 8), (1, 4, 1, 8), (4, 5, 8), (5, 8), (3, 1, 5, 8), (3, 4, 5, 1), (7,), (1, 3, 4, 5, 8), ()):
        with pytest.raises(ValueError):
            N._gate(torch.zeros(shape), b)


def test_dense_memory_in_any_order():
    from lookatmyquant_b200 import gradients as G
    x = torch.zeros(4, 5, 6)
    for y in (x, x.permute(2, 0, 1), x[1:3], x[:, :, :1].contiguous(), x[:1], torch.zeros(()), torch.zeros(3, 0), x.mT[:, 0:0]):
        assert G._dense(y)
    for y in (x[:, 1:], x[..., ::2], torch.zeros(5).expand(4, 5), x[:, 0], x.mT[:, 1:]):
        assert not G._dense(y)


def test_lists_are_refused_before_the_device_is_asked():
    from lookatmyquant_b200 import gradients as G
    for call, error in ((lambda: G.global_norm([]), ValueError), (lambda: G.global_norm([None]), ValueError),
                        (lambda: G.global_norm([torch.zeros(3)]), TypeError), (lambda: G.global_norm([1.0]), TypeError),
                        (lambda: G.clip([torch.zeros(3)], 1.0), TypeError), (lambda: G.clip([None], 1.0, []), ValueError)):
        with pytest.raises(error):
            call()
