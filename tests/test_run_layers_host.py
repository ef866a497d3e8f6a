"""norms.run_layers on small random Hugging Face models without a GPU: the model's own masks, multipliers and norms, or a refusal.

torch forms of `norm` and `join` stand in, written in the models' own order of operations, so that what is right is equal bit
for bit to the model's own forward.
"""

import pytest
import torch

transformers = pytest.importorskip("transformers")


def plain_norm(x, weight, eps=1e-6, offset=0.0):
    assert offset == 0.0
    f = x.to(torch.float32)
    f = f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + eps)
    return weight * f.to(x.dtype)


def plain_join(residual, branch, weight=None, post_weight=None, gate=None, scale=1.0, eps=1e-6, offset=0.0):
    assert gate is None
    if post_weight is not None:
        branch = plain_norm(branch, post_weight, eps, offset)
    h = residual + (branch if scale == 1.0 else branch * scale)
    return h, None if weight is None else plain_norm(h, weight, eps, offset)


@pytest.fixture
def N(monkeypatch):
    from lookatmyquant_b200 import norms
    monkeypatch.setattr(norms, "norm", plain_norm)
    monkeypatch.setattr(norms, "join", plain_join)
    return norms


def build(name, attention="sdpa", **kw):
    torch.manual_seed(3)
    heads = {} if name == "Granite" else {"head_dim": 8}
    config = getattr(transformers, name + "Config")(
        hidden_size=32, intermediate_size=48, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, vocab_size=64,
        pad_token_id=0, attn_implementation=attention, **heads, **kw)
    model = transformers.AutoModelForCausalLM.from_config(config).eval()
    with torch.no_grad():
        for p in model.parameters():
            p.add_(torch.randn_like(p) * 0.3)  # norms whose weights are not one, attention that is not flat
    return model


RIGHT = [("Llama", {}), ("Qwen2", {}), ("Qwen3", {}), ("Qwen3", {"num_hidden_layers": 0}),
         ("Mistral", {"sliding_window": 4}), ("Qwen2", {"use_sliding_window": True, "sliding_window": 5, "max_window_layers": 1}),
         ("Granite", {"residual_multiplier": 0.22, "embedding_multiplier": 3.0, "logits_scaling": 8.0,
                      "attention_multiplier": 0.3}),
         ("Glm4", {}), ("Phi3", {"resid_pdrop": 0.0})]


@pytest.mark.parametrize("attention", ["sdpa", "eager"])
@pytest.mark.parametrize("name,kw", RIGHT, ids=[f"{n}-{i}" for i, (n, _) in enumerate(RIGHT)])
def test_states_and_gradients_are_the_models_own(N, name, kw, attention):
    layers = {"num_hidden_layers": 3, **kw}
    kw = {k: v for k, v in kw.items() if k != "num_hidden_layers"}
    model = build(name, attention, **kw)
    if not layers["num_hidden_layers"]:
        model.model.layers = model.model.layers[:0]
        model.config.num_hidden_layers = 0
    x = torch.randn(2, 13, 32)
    results = []
    for run in (lambda e: model.model(inputs_embeds=e, use_cache=False).last_hidden_state, lambda e: N.run_layers(model, e)):
        model.zero_grad(set_to_none=True)
        e = x.clone().requires_grad_(True)
        out = run(e)
        out.square().sum().backward()
        results.append((out.detach(), e.grad, {n: p.grad for n, p in model.named_parameters()}))
    (want, dx, grads), (got, dy, other) = results
    assert torch.equal(got, want)
    assert torch.equal(dy, dx)
    for n, g in grads.items():
        assert (g is None) == (other[n] is None) and (g is None or torch.equal(other[n], g)), n


def test_the_model_is_left_as_it_was(N):
    model = build("Llama")
    before = {n: id(m) for n, m in model.named_modules()}
    keys = [set(vars(m)) for m in model.modules()]
    N.run_layers(model, torch.randn(1, 5, 32))
    assert before == {n: id(m) for n, m in model.named_modules()} and keys == [set(vars(m)) for m in model.modules()]


def test_a_default_type_changes_no_norm(N):
    """A class's formula is found out once, in fp32 whatever torch's default is then."""
    from lookatmyquant_b200 import decoder
    decoder._is_rms.cache_clear()
    model, x = build("Llama"), torch.randn(1, 5, 32)
    want = model.model(inputs_embeds=x, use_cache=False).last_hidden_state
    torch.set_default_dtype(torch.bfloat16)
    try:
        got = N.run_layers(model, x)
    finally:
        torch.set_default_dtype(torch.float32)
        decoder._is_rms.cache_clear()
    assert torch.equal(got, want)


def test_a_model_may_name_the_states(N):
    model = build("Llama")

    class Named(type(model.model)):
        def forward(self, inputs_embeds=None, use_cache=None):
            h = inputs_embeds
            kw = dict(attention_mask=None, position_embeddings=self.rotary_emb(h, torch.arange(h.shape[1])[None]))
            for layer in self.layers:
                h = layer(hidden_states=h, **kw)
            return transformers.modeling_outputs.BaseModelOutputWithPast(last_hidden_state=self.norm(h))
    model.model.__class__ = Named
    x = torch.randn(2, 5, 32)
    assert torch.equal(N.run_layers(model, x), model.model(inputs_embeds=x).last_hidden_state)


def test_hooks_of_what_still_runs_are_called(N):
    model, seen = build("Llama"), []
    for n, m in model.named_modules():
        if n.endswith(("self_attn", "mlp", "q_proj", "rotary_emb")) or n == "model":
            m.register_forward_hook(lambda *_, n=n: seen.append(n))
    N.run_layers(model, torch.randn(1, 5, 32))
    assert len(seen) == 2 + 3 * 3


class Scaled(torch.nn.Module):
    """A norm of the same attributes and another formula."""

    def __init__(self, like):
        super().__init__()
        self.weight, self.variance_epsilon = like.weight, like.variance_epsilon

    def forward(self, x):
        return (1 + self.weight) * torch.nn.functional.rms_norm(x, x.shape[-1:], None, self.variance_epsilon)


def changed(f):
    model = build("Llama")
    f(model)
    return model


def hook(module):
    module.register_forward_hook(lambda *_: None)


def before_hook(module):
    module.register_full_backward_hook(lambda *_: None)


def norm_after(layer):
    """A layer of the same children that norms what its blocks give, and not what they take."""
    def forward(h, **kw):
        h = h + layer.input_layernorm(layer.self_attn(hidden_states=h, **kw)[0])
        return h + layer.post_attention_layernorm(layer.mlp(h))
    return forward


def swapped(model):
    class Other(type(model.model.layers[0])):
        def forward(self, h, **kw):
            h = h + self.input_layernorm(self.self_attn(hidden_states=h, **kw)[0])
            return h + self.post_attention_layernorm(self.mlp(h))
    model.model.layers[1].__class__ = Other


def checkpointed(model):
    model.gradient_checkpointing_enable()
    model.train()


def biased(model):
    model.model.layers[0].input_layernorm = torch.nn.LayerNorm(32)


REFUSED = [
    (TypeError, lambda: build("Gemma")), (TypeError, lambda: build("Olmo2")),
    (TypeError, lambda: changed(swapped)), (TypeError, lambda: changed(biased)),
    (TypeError, lambda: changed(lambda m: setattr(m.model.layers[0], "forward", norm_after(m.model.layers[0])))),
    (TypeError, lambda: changed(lambda m: setattr(m.model, "norm", Scaled(m.model.norm)))),
    (TypeError, lambda: changed(lambda m: setattr(m.model.layers[2], "input_layernorm", Scaled(m.model.norm)))),
    (TypeError, lambda: torch.nn.Linear(32, 32)),
    (ValueError, lambda: changed(checkpointed)), (ValueError, lambda: changed(lambda m: hook(m.model.layers[1]))),
    (ValueError, lambda: changed(lambda m: hook(m.model.layers[1].input_layernorm))),
    (ValueError, lambda: changed(lambda m: hook(m.model.norm))),
    (ValueError, lambda: changed(lambda m: before_hook(m.model.layers[2].post_attention_layernorm))),
    (ValueError, lambda: changed(lambda m: before_hook(m.model.layers[2]))),
    (ValueError, lambda: build("Phi3", resid_pdrop=0.1).train()),
]


@pytest.mark.parametrize("error,make", REFUSED, ids=range(len(REFUSED)))
def test_other_layers_are_refused(N, error, make):
    with pytest.raises(error, match="run_layers|joined"):
        N.run_layers(make(), torch.randn(1, 5, 32))
