"""The training operators together: as a transformers model's attention, under row importance's backward pass, and in a
fine-tuning run. Against the same model in fp32 (eager attention) the bf16 model's outputs and gradients on these kernels
may be off by what torch's own bf16 attention is off, and half as much again (both round to bf16 everywhere else)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def models():
    from transformers import LlamaForCausalLM

    from lookatmyquant_b200 import attention, measure
    attention.use_in_transformers()
    lamq = measure.build_model(2, attention="lamq")
    sdpa = measure.build_model(2)
    cfg = measure.smollm2_config(2, "eager")
    exact = LlamaForCausalLM(cfg)
    exact.load_state_dict(sdpa.state_dict())
    return lamq, sdpa, exact.cuda().float().eval()


def gradients(model, ids):
    model.zero_grad(set_to_none=True)
    out = model(ids, use_cache=False).logits.float()
    torch.log_softmax(out, -1).gather(-1, ids.roll(-1, 1)[..., None]).mean().neg().backward()
    got = {n: p.grad.double() for n, p in model.named_parameters()}
    model.zero_grad(set_to_none=True)
    return out.detach().double(), got


def test_model_outputs_and_gradients(models):
    from lookatmyquant_b200 import measure
    ids = measure.zipf_tokens(2, 333, 49152, 5).cuda()
    (yl, gl), (ys, gs), (ye, ge) = (gradients(m, ids) for m in models)
    off = lambda x, e: float((x - e).norm() / e.norm())
    assert off(yl, ye) <= 1.5 * off(ys, ye)
    for name in ge:
        assert off(gl[name], ge[name]) <= 1.5 * off(gs[name], ge[name]) + 1e-4, name


def test_row_importance_runs_on_the_kernels(models):
    from lookatmyquant_b200 import importance, measure
    ids = measure.zipf_tokens(1, 200, 49152, 6)
    imp = {}
    for key, model in zip(("lamq", "sdpa", "exact"), models):
        mods = {"q": model.model.layers[0].self_attn.q_proj, "v": model.model.layers[1].self_attn.v_proj}
        imp[key] = importance.row_importance(model, ids, mods, sampled=[ids[0]])[0]
    for name in ("q", "v"):
        e = imp["exact"][name]
        assert float((imp["lamq"][name] - e).norm()) <= 1.5 * float((imp["sdpa"][name] - e).norm()) + 1e-3 * float(e.norm())


def test_masks_that_are_not_whole_windows_are_refused(models):
    ids = torch.arange(20, device="cuda").reshape(2, 10)
    mask = torch.ones_like(ids)
    whole = models[0](ids, attention_mask=mask, use_cache=False).logits
    assert torch.equal(whole, models[0](ids, use_cache=False).logits)
    mask[0, :3] = 0
    with pytest.raises(NotImplementedError):
        models[0](ids, attention_mask=mask, use_cache=False)


def test_cached_generation_sees_all_keys(models):
    """One token after a cached prefix gets the logits of the whole window's last position."""
    ids = torch.arange(40, 61, device="cuda")[None]
    with torch.no_grad():
        past = models[0](ids[:, :-1], use_cache=True).past_key_values
        last = models[0](ids[:, -1:], past_key_values=past, use_cache=True).logits[0, -1].double()
        full = models[0](ids, use_cache=False).logits[0, -1].double()
    assert float((last - full).norm() / full.norm()) <= 2.0**-6


def test_tuning_learns_its_windows():
    """The loss starts at about log(vocabulary) (a random model) and falls by a third in 8 steps on 400 tokens; the first
    losses of two runs agree bit for bit."""
    from lookatmyquant_b200 import tune
    losses = tune.run(layers=2, windows=2, T=201, steps=8, log=lambda s: None)
    assert 10.0 < losses[0] < 12.5 and losses[-1] < 0.67 * losses[0], losses
    assert tune.run(layers=2, windows=2, T=201, steps=1, log=lambda s: None)[0] == losses[0]
