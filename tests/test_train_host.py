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
