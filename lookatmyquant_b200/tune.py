"""Fine-tuning a model around its coded matrices, end to end on this package's kernels: the scaled embedding lookup and
its gradient (embedding.scaled_embedding), attention forwards and backwards (attention.attention, as the model's
attention implementation) and Muon updates (orthogonal.Muon) of the matrices that are still free; on request the layers'
norms joined with their residual additions (decoder.joined, as norms.run_layers does) and the gradients clipped by their
global norm (gradients.clip).

The student is the model with some of its matrices replaced by their trellis words (here: every down_proj, as `measure`
codes a piece); those stay. The loss is the mean cross-entropy of the windows' next tokens; Muon moves the free matrices,
plain gradient descent the embedding table. The model is a random-initialised SmolLM2-360M-architecture Llama and the
windows are seeded Zipf tokens, as in `measure`.

    python -m lookatmyquant_b200.tune [--layers 2] [--windows 4] [--T 256] [--steps 8] [--option tr2] [--fused-norms]
                                      [--clip 1.0]
"""

from __future__ import annotations

import torch

from . import attention, codes, decoder, embedding, gradients, orthogonal
from .measure import BLOCK_SEED, build_model, capture, zipf_tokens

FREE = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj")


def coded(model, option: str, chunks: list) -> list:
    """Replaces every down_proj's weight by its trellis word's at `option` (tr1..tr4) under the stage's statistics, as
    `measure` does for a piece, and freezes it. Returns the words."""
    words = []
    kbits = int(option[2:])
    for i, layer in enumerate(model.model.layers):
        H = capture(model, [i], chunks)[(i, "mlp.down_proj")]
        W = layer.mlp.down_proj.weight
        Tm = next(t for t in (320, 256, 128, 64) if W.shape[0] % t == 0)
        word = codes.ldlq_words([W.double()], H, codes.TrellisCode(12, kbits, T=Tm), [1000 * i + 100 * BLOCK_SEED["mlp"]])[0]
        W.data = word.matrix().to(W.dtype)
        W.requires_grad_(False)
        words.append(word)
    return words


class Tuner:
    """A student model, the free parameters and their optimisers; `step(ids)` is one update. `fused_norms` runs the model
    through decoder.joined; with `max_norm` the gradients of all free parameters together are clipped to it, and
    `grad_norm` is their norm before (a scalar on the device)."""

    def __init__(self, model, lr: float = 0.02, table_lr: float = 0.02, scale: float = 1.0, fused_norms: bool = False,
                 max_norm: float | None = None):
        self.model, self.scale, self.table_lr = model, scale, table_lr
        self.fused_norms, self.max_norm, self.grad_norm = fused_norms, max_norm, None
        self.table = model.get_input_embeddings().weight
        for p in model.parameters():
            p.requires_grad_(False)
        free = [p for name, p in model.named_parameters() if name.split(".")[-2] in FREE]
        self.free = [*free, self.table]
        for p in self.free:
            p.requires_grad_(True)
        self.muon = orthogonal.Muon(free, lr=lr)

    def logits(self, ids: torch.Tensor) -> torch.Tensor:
        """The student's logits: the table's rows looked up (scaled), the layers, the model's own head."""
        x = embedding.scaled_embedding(self.table, ids, self.scale)
        model = decoder.joined(self.model) if self.fused_norms else self.model
        return model(inputs_embeds=x, use_cache=False).logits

    def loss(self, ids: torch.Tensor) -> torch.Tensor:
        """The mean cross-entropy of the windows' next tokens."""
        return torch.nn.functional.cross_entropy(self.logits(ids[:, :-1]).float().flatten(0, 1), ids[:, 1:].flatten())

    def step(self, ids: torch.Tensor) -> float:
        loss = self.loss(ids)
        self.muon.zero_grad(set_to_none=True)
        self.table.grad = None
        loss.backward()
        if self.max_norm is not None:
            self.grad_norm = gradients.clip([p.grad for p in self.free], self.max_norm)
        self.muon.step()
        with torch.no_grad():
            self.table.add_(self.table.grad, alpha=-self.table_lr)
        return float(loss.detach())

    def check_status(self):
        """Raises if a kernel of any step reported an error."""
        for module in (attention, embedding, orthogonal):
            module.check_status()


def run(layers: int = 2, windows: int = 4, T: int = 256, steps: int = 8, option: str = "tr2", lr: float = 0.02,
        seed: int = 0, device="cuda", log=print, fused_norms: bool = False, max_norm: float | None = None) -> list:
    """Codes the down_projs, then `steps` updates on the same windows (`fused_norms`, `max_norm`: as the Tuner's). Returns the
    loss before each and after the last."""
    model = build_model(layers, seed, device, attention=attention.use_in_transformers())
    ids = zipf_tokens(windows, T, model.config.vocab_size, seed + 1).to(device)
    with torch.no_grad():
        coded(model, option, [ids])
    tuner = Tuner(model, lr=lr, fused_norms=fused_norms, max_norm=max_norm)
    losses = [tuner.step(ids) for _ in range(steps)]
    with torch.no_grad():
        losses.append(float(tuner.loss(ids)))
    tuner.check_status()
    for k, x in enumerate(losses):
        log(f"  step {k}: loss {x:.4f}")
    return losses


def main():
    """`python -m lookatmyquant_b200.tune`: codes every down_proj of a random SmolLM2-360M-architecture model and tunes
    the rest of it on the windows' next tokens; prints the loss of every step."""
    import argparse
    ap = argparse.ArgumentParser(description=main.__doc__)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--windows", type=int, default=4)
    ap.add_argument("--T", type=int, default=256)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--option", default="tr2")
    ap.add_argument("--lr", type=float, default=0.02)
    ap.add_argument("--fused-norms", action="store_true", help="the layers' norms joined with their residual additions")
    ap.add_argument("--clip", type=float, metavar="NORM", help="clip the gradients to this global norm")
    a = ap.parse_args()
    run(a.layers, a.windows, a.T, a.steps, a.option, a.lr, fused_norms=a.fused_norms, max_norm=a.clip)


if __name__ == "__main__":
    main()
