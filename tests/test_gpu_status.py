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
