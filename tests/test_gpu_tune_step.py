"""The norms and the clipping as a fine-tuning step uses them, with attention, embedding and Muon beside them."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def models():
    """The same random weights: bf16 on the package's attention, and fp32 with torch's own everything."""
    from transformers import LlamaForCausalLM

    from lookatmyquant_b200 import attention, measure
    model = measure.build_model(3, attention=attention.use_in_transformers())
    exact = LlamaForCausalLM(measure.smollm2_config(3, "eager"))
    exact.load_state_dict(model.state_dict())
    return model, exact.cuda().float().eval()


def gradients_of(model, logits, ids):
    model.zero_grad(set_to_none=True)
    torch.log_softmax(logits.float(), -1).gather(-1, ids.roll(-1, 1)[..., None]).mean().neg().backward()
    got = {n: p.grad.double() for n, p in model.named_parameters()}
    model.zero_grad(set_to_none=True)
    return got


def test_a_model_runs_on_the_joined_norms(models):
    """Outputs and all gradients, the norms' weights' among them: against fp32 off by what the model's own bf16 norms and
    additions are off, and half as much again (the joins round once where those round twice)."""
    from lookatmyquant_b200 import measure, norms
    model, exact = models
    ids = measure.zipf_tokens(2, 333, 49152, 5).cuda()
    plain = model(ids, use_cache=False).logits
    joined = model.lm_head(norms.run_layers(model, model.get_input_embeddings()(ids)))
    want = exact(ids, use_cache=False).logits
    off = lambda x, e: float((x.detach().double() - e.detach()).norm() / e.detach().norm())
    assert off(joined, want.double()) <= 1.5 * off(plain, want.double())
    ge = gradients_of(exact, want, ids)
    gp, gj = gradients_of(model, plain, ids), gradients_of(model, joined, ids)
    for name in ge:
        assert off(gj[name], ge[name]) <= 1.5 * off(gp[name], ge[name]) + 1e-4, name


def test_a_tuning_step_clips_its_gradients():
    """The gradients that Muon and the table's descent see have the bound's norm, the reported norm is the one before; a bound
    that is never met changes no bit of a run, and steps run with everything on."""
    from lookatmyquant_b200 import attention, gradients, measure, tune
    ids = measure.zipf_tokens(2, 129, 49152, 7).cuda()

    def tuner(**kw):
        return tune.Tuner(measure.build_model(1, attention=attention.use_in_transformers()), **kw)
    free = tuner()
    first = free.step(ids)
    before = float(gradients.global_norm([p.grad for p in free.free]))
    same = tuner(max_norm=10 * before)
    assert same.step(ids) == first and float(same.grad_norm) == before
    assert all(torch.equal(a, b) for a, b in zip(free.free, same.free))
    tight = tuner(max_norm=before / 50, fused_norms=True)
    for _ in range(2):
        assert math.isfinite(tight.step(ids))
        after = float(gradients.global_norm([p.grad for p in tight.free]))
        # every element rounded to bf16 (at most 2^-8 of it), and the factor
        assert float(tight.grad_norm) > before / 25 and abs(after * 50 / before - 1) <= 2.0**-8 + 1e-5
    tight.check_status()


def test_the_command_takes_both(capsys, monkeypatch):
    from lookatmyquant_b200 import tune
    monkeypatch.setattr("sys.argv", ["tune", "--layers", "1", "--windows", "1", "--T", "65", "--steps", "1", "--fused-norms",
                                     "--clip", "0.5"])
    tune.main()
    assert "step 1: loss" in capsys.readouterr().out


def test_a_whole_step_in_one_graph():
    """norm, join, their gradients, the global norm and the clipping captured together and replayed on new inputs."""
    from lookatmyquant_b200 import gradients, norms
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.randn(4, 50, 320, device="cuda", generator=g).bfloat16()
    w = [torch.randn(320, device="cuda", generator=g).bfloat16() for _ in range(2)]

    def step():
        y = norms.norm_forward(x, w[0])
        h, z = norms.join_forward(x, y, w[1], post_weight=w[0], scale=0.5)
        dr, db, dw, du, _ = norms.join_backward(h, z, h, y, w[1], post_weight=w[0], scale=0.5)
        dx, dv = norms.norm_backward(db, x, w[0])
        return gradients.clip([dr, dx, dw, du, dv], 1.0), dr, dx, dw, du, dv
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        x.copy_(torch.randn(x.shape, device="cuda", generator=g))
        graph.replay()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
