"""Models of other masks, multipliers and norms than the package's own on the joined norms: against fp32, bf16 states and gradients
are off by what the model's own bf16 forward is off, and half as much again (a join rounds once where that rounds twice or
more; what it cannot see, a mask or a multiplier left out, is off by tens of percents)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

MODELS = [("Llama", {}), ("Mistral", {"sliding_window": 16}), ("Granite", {"residual_multiplier": 0.22, "logits_scaling": 8.0}),
          ("Glm4", {})]


def off(x, exact):
    x, exact = x.detach().double(), exact.detach().double()
    return float((x - exact).norm() / exact.norm())


@pytest.mark.parametrize("attention", ["sdpa", "eager"])
@pytest.mark.parametrize("name,kw", MODELS, ids=[m[0] for m in MODELS])
def test_the_models_own_masks_and_multipliers(name, kw, attention):
    import transformers

    from lookatmyquant_b200 import norms
    torch.manual_seed(5)
    heads = {} if name == "Granite" else {"head_dim": 64}
    config = getattr(transformers, name + "Config")(
        hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, vocab_size=512,
        pad_token_id=0, attn_implementation=attention, **heads, **kw)
    exact = transformers.AutoModelForCausalLM.from_config(config).eval().cuda()
    with torch.no_grad():
        for p in exact.parameters():
            p.copy_((p + 0.05 * torch.randn_like(p)).bfloat16())
    model = transformers.AutoModelForCausalLM.from_config(config).eval().cuda()
    model.load_state_dict(exact.state_dict())
    model.bfloat16()
    x = torch.randn(2, 77, 256, device="cuda").bfloat16()
    ds = torch.randn(2, 77, 256, device="cuda").bfloat16()

    def run(m, forward, dtype):
        m.zero_grad(set_to_none=True)
        e = x.to(dtype).requires_grad_(True)
        out = forward(m, e)
        out.backward(ds.to(dtype))
        grads = torch.cat([p.grad.flatten().double() for p in m.model.layers.parameters()])
        return out, e.grad, grads
    own = lambda m, e: m.model(inputs_embeds=e, use_cache=False).last_hidden_state
    want, plain = run(exact, own, torch.float32), run(model, own, torch.bfloat16)
    got = run(model, norms.run_layers, torch.bfloat16)
    for g, p, w in zip(got, plain, want):
        assert off(g, w) <= 1.5 * off(p, w)
