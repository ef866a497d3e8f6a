"""Updates orthogonalised by Newton-Schulz products, and the Muon optimiser that takes them, on B200 (liblamq_b200:
lamq_newton_schulz).

Fine-tuning moves a model's matrices (the ones this package codes, or the ones between them) by gradients whose few
strong directions drown the others. Muon's update is the momentum with its singular values taken to about 1: an odd
polynomial iterated in the matrix, products only. All iterations run in one kernel on the tensor cores, in fp16 pairs
(22 bits) where rounding would grow and fp16 where it cannot; the result is bf16.
"""

from __future__ import annotations

import functools
import math
import struct

import torch

from . import _lib
from ._lib import check, launch_on, ptr

COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # Muon's quintic: steep at zero, singular values end within about [0.7, 1.2]

_STATUS = _lib.StatusWord("newton_schulz")
_DTYPES = {torch.float32: _lib.LAMQ_F32, torch.bfloat16: _lib.LAMQ_BF16}


def check_status():
    """Raises if a kernel of any call so far gave up on a device wait (its results are then invalid). Waits for the
    device."""
    _STATUS.check()


@functools.lru_cache(maxsize=64)
def _coefficients(coefficients: tuple, steps: int) -> bytes:
    rows = coefficients if isinstance(coefficients[0], tuple) else (coefficients,) * steps
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError("coefficients: one (a, b, c), or one for each step")
    return struct.pack(f"{3 * steps}f", *(x for r in rows for x in r))


def newton_schulz(G: torch.Tensor, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7) -> torch.Tensor:
    """G (..., m, n; fp32 or bf16) orthogonalised: X = G / (|G|_F + eps), then `steps` times X <- (aI + bA + cA²)X with
    A = X·Xᵀ (on the smaller side). `coefficients` is one (a, b, c) or a sequence of one per step; 1 to 16 steps. bf16, G's
    shape; the matrices of a batch go together in one launch.

    X and the polynomials are held in fp16 pairs, so coefficients raise ValueError where they can take a singular value of
    [0, 1] above 5, or |a + b·s² + c·s⁴| above 32, in any step. Steps steeper than 9 anywhere (Muon's: 4) take 2.6 times the
    products, for the same error."""
    if G.dtype not in _DTYPES or not G.is_cuda:
        raise TypeError("the update must be a float32 or bfloat16 CUDA tensor")
    if G.ndim < 2:
        raise ValueError("the update must be a matrix or a batch of matrices")
    if not isinstance(coefficients, tuple) or not all(isinstance(c, (float, tuple)) for c in coefficients):
        coefficients = tuple(tuple(map(float, c)) if hasattr(c, "__len__") else float(c) for c in coefficients)
    coef = _coefficients(coefficients, steps) if steps > 0 else b""
    m, n = G.shape[-2:]
    dev = G.device
    X = G if G.ndim <= 3 else G.reshape(math.prod(G.shape[:-2]), m, n)
    batch = X.shape[0] if X.ndim == 3 else 1
    if X.numel() and (X.stride(-1) != 1 or (m > 1 and X.stride(-2) < n) or
                      (batch > 1 and X.stride(0) < (m - 1) * X.stride(-2) + n)):
        X = X.contiguous()
    out = torch.empty(G.shape, dtype=torch.bfloat16, device=dev)
    lib = _lib.load()
    ws = torch.empty(lib.lamq_newton_schulz_workspace_size(batch, m, n), dtype=torch.uint8, device=dev)
    here, stream = launch_on(dev)
    with here:
        check(lib.lamq_newton_schulz(ptr(X), _DTYPES[X.dtype], max(X.stride(-2), n) if X.numel() else n,
                                     X.stride(0) if X.ndim == 3 else 0, batch, m, n, steps, coef, eps, ptr(out),
                                     ptr(ws), ws.numel(), ptr(_STATUS.on(dev)), stream), "lamq_newton_schulz")
    return out


class Muon(torch.optim.Optimizer):
    """Momentum whose update is orthogonalised, for matrices (..., m, n): with g the gradient and b the momentum buffer
    (fp32), b <- momentum·b + g, u = g + momentum·b (Nesterov) or b, and
    p <- p·(1 − lr·weight_decay) − lr·sqrt(max(1, m/n))·newton_schulz(u). Parameters of one shape go to the kernel as a
    batch."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 steps: int = 5, coefficients=COEFFICIENTS):
        if lr < 0 or not 0 <= momentum < 1 or weight_decay < 0:
            raise ValueError("lr and weight_decay must not be negative, momentum in [0, 1)")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      steps=steps, coefficients=coefficients))
        for group in self.param_groups:
            if any(p.ndim < 2 for p in group["params"]):
                raise ValueError("Muon updates matrices: leave vectors to another optimiser")

    def load_state_dict(self, state_dict):
        """As every optimiser's, with the momentum kept in fp32 (torch casts state to the parameters' type)."""
        super().load_state_dict(state_dict)
        saved = (key for group in state_dict["param_groups"] for key in group["params"])
        for key, p in zip(saved, (p for group in self.param_groups for p in group["params"])):
            momentum = state_dict["state"].get(key, {}).get("momentum")
            if momentum is not None:
                self.state[p]["momentum"] = momentum.detach().to(p.device, torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            shapes = {}
            for p in group["params"]:
                if p.grad is not None:
                    shapes.setdefault((p.shape, p.device), []).append(p)
            mu = group["momentum"]
            for params in shapes.values():
                us = []
                for p in params:
                    state = self.state[p]
                    if "momentum" not in state:
                        state["momentum"] = torch.zeros_like(p, dtype=torch.float32)
                    b, g = state["momentum"], p.grad.float()
                    b.mul_(mu).add_(g)
                    us.append(torch.add(g, b, alpha=mu) if group["nesterov"] else b)
                O = newton_schulz(us[0] if len(us) == 1 else torch.stack(us), group["steps"], group["coefficients"])
                m, n = params[0].shape[-2:]
                rate = -group["lr"] * max(1.0, m / max(n, 1)) ** 0.5
                for p, o in zip(params, (O,) if len(us) == 1 else O.unbind(0)):
                    if group["weight_decay"]:
                        p.mul_(1.0 - group["lr"] * group["weight_decay"])
                    p.add_(o, alpha=rate)
        return loss
