"""The tuner's logits with and without the joined norms, without a GPU: whatever a model does behind its layers is in both."""

import pytest
import torch
from test_run_layers_host import N, build  # noqa: F401  (N: torch forms of norm and join stand in)


@pytest.mark.parametrize("name,kw", [("Llama", {}), ("Granite", {"logits_scaling": 8.0, "embedding_multiplier": 3.0})])
def test_fused_norms_change_no_logit(N, monkeypatch, name, kw):  # noqa: F811
    from lookatmyquant_b200 import embedding, orthogonal, tune
    monkeypatch.setattr(embedding, "scaled_embedding", lambda table, ids, scale: scale * table[ids])
    monkeypatch.setattr(orthogonal, "Muon", lambda params, lr: None)
    model = build(name, **kw)
    ids = torch.arange(26).view(2, 13)
    want = tune.Tuner(model).logits(ids)
    got = tune.Tuner(model, fused_norms=True).logits(ids)
    assert torch.equal(got, want)
