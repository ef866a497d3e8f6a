"""Further measured cases of the training operators: the norms around a block (alone, and joined with the residual
addition, its gate and its scale), forwards and backwards, and the global norm of many gradients with its clipping.

`listed()` gives the cases, `draw(rng)` one more of the same ranges, `prepare(case, seed)` the tensors that a training
loop holds before the call, `run(state)` one call (`own` false: elementary fp32 torch operations; true: the package's
operators), `work(case)` the bytes and operations that the call cannot do without, and `exact(case, seed)` its result
in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
CLIP_EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------------- cases

def _norm(op, B, L, H, d, dtype="bf16", offset=0.0):
    """H > 1: the heads of a projection whose output also holds other heads (the rows are strided)."""
    return {"op": op, "B": B, "L": L, "H": H, "d": d, "dtype": dtype, "offset": offset}


def _join(op, B, L, d, residual="bf16", branch="bf16", post=False, gate="none", scale=1.0, pre=True):
    return {"op": op, "B": B, "L": L, "d": d, "residual": residual, "branch": branch, "post": post, "gate": gate,
            "scale": scale, "pre": pre}


def _gradients(op, layers, hidden, kv, mlp, vocab, dtype="bf16", out="none", within=False):
    """The gradients of a model's matrices and norms; `out`: the type of separate buffers for the clipped ones ("none":
    in place); `within`: the norm is below the bound."""
    return {"op": op, "layers": layers, "hidden": hidden, "kv": kv, "mlp": mlp, "vocab": vocab, "dtype": dtype, "out": out,
            "within": within}


def listed():
    cases = [
        # the final norm of one token (the smallest call: latency)
        ("norm one token", _norm("norm", 1, 1, 1, 960)),
        # the query heads of four long windows, normed in place in the output of the joint q, k, v projection
        ("norm query heads", _norm("norm", 4, 2048, 32, 128)),
        # the gradient of one short text: row importance over single calibration texts
        ("norm backward 77 tokens", _norm("norm_backward", 1, 77, 1, 960)),
        # a fine-tuning step's windows through a 2560-wide model
        ("norm backward windows", _norm("norm_backward", 8, 2048, 1, 2560)),
        # one token through a block of a 960-wide model
        ("join one token", _join("join", 1, 1, 960)),
        # norms before and after the block, a gate for each text, an fp32 residual stream
        ("join sandwich", _join("join", 2, 4096, 2560, "fp32", "bf16", True, "text", 0.22)),
        # ragged and odd: rows that start anywhere, a gate for each element, everything fp32
        ("join backward odd", _join("join_backward", 5, 667, 1337, "fp32", "fp32", True, "token", 0.5)),
        # the largest step: norms on both sides and a learned gate per channel
        ("join backward sandwich", _join("join_backward", 2, 4096, 4096, "bf16", "bf16", True, "channel", 1.0)),
        # the norm that a tuning run of a two-layer model logs
        ("global norm two layers", _gradients("global_norm", 2, 960, 320, 2560, 49152)),
        # the same for four 2560-wide layers with fp32 gradients
        ("global norm four layers", _gradients("global_norm", 4, 2560, 1024, 9728, 0, "fp32")),
        # most steps: the norm is within the bound, nothing changes
        ("clip within the bound", _gradients("clip", 2, 960, 320, 2560, 49152, "bf16", "none", True)),
        # a step that is clipped, fp32 gradients into buffers of their own
        ("clip four layers", _gradients("clip", 4, 2560, 1024, 9728, 0, "fp32", "fp32")),
    ]
    return [{"name": name, **case} for name, case in cases]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["norm", "norm_backward", "join", "join", "join_backward", "join_backward", "global_norm", "clip"])
    most = 2 * 4096 * 4096
    if op.startswith("norm"):
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        if rng.random() < 0.3:
            H, d = rng.choice([(15, 64), (32, 128), (5, 64), (6, 80), (7, 33)])
        else:
            H, d = 1, rng.choice([960, 1000, 2560, 4096, 9728, _log_int(rng, 16, 8192), _log_int(rng, 16, 8192)])
        n = _log_int(rng, 1, min(65536, most // (H * d)))
        B = rng.choice([1, 1, 2, 5])
        return _norm(op, B, max(1, n // B), H, d, dtype, rng.choice([0.0, 0.0, 1.0]))
    if op.startswith("join"):
        d = rng.choice([960, 1000, 2560, 4096, 9728, _log_int(rng, 16, 8192), _log_int(rng, 16, 8192)])
        residual, branch = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("fp32", "bf16"), ("fp32", "fp32")])
        n = _log_int(rng, 1, min(65536, most // d // (1 if residual == branch == "bf16" else 2)))
        B = rng.choice([1, 2, 3, 8])
        return _join(op, B, max(1, n // B), d, residual, branch, rng.random() < 0.5,
                     rng.choice(["none", "none", "channel", "text", "token"]), rng.choice([1.0, 0.22]),
                     rng.random() < 0.85)
    hidden = _log_int(rng, 33, 2560)
    layers, mlp = rng.randint(1, 4), _log_int(rng, hidden, 3 * hidden)
    out = rng.choice(["none", "bf16", "fp32"]) if op == "clip" else "none"
    # in place only within the bound: a pass that clips would leave the next one another input
    return _gradients(op, layers, hidden, max(1, hidden // rng.choice([1, 3, 4])), mlp,
                      rng.choice([0, _log_int(rng, 256, 49152)]), rng.choice(["bf16", "fp32"]), out, out == "none")


# --------------------------------------------------------------------------------------------------------------- inputs

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _shapes(case):
    d, kv, mlp = case["hidden"], case["kv"], case["mlp"]
    layer = [(d, d), (kv, d), (kv, d), (d, d), (mlp, d), (mlp, d), (d, mlp), (d,), (d,)]
    return layer * case["layers"] + ([(case["vocab"], d)] if case["vocab"] else [])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def stream(*shape):  # activations: a scale per channel, a few of them far above the rest
        d = shape[-1]
        channels = torch.exp(0.5 * normal(d)) * torch.where(torch.rand(d, device="cuda", generator=g) < 0.003, 20.0, 1.0)
        return normal(*shape) * channels

    if case["op"].startswith("norm"):
        B, L, H, d, dt = case["B"], case["L"], case["H"], case["d"], _TYPES[case["dtype"]]
        if H > 1:  # some more heads behind these in the projection's output
            x = stream(B, L, (H + H // 2) * d).to(dt).view(B, L, H + H // 2, d)[:, :, :H]
        else:
            x = stream(B, L, d).to(dt)
        st = {"case": case, "x": x, "weight": ((1.0 - case["offset"]) + 0.1 * normal(d)).to(dt)}
        if case["op"] == "norm_backward":
            st["dy"] = (1e-3 * normal(*x.shape)).to(dt)
        return st
    if case["op"].startswith("join"):
        B, L, d, dr, db = case["B"], case["L"], case["d"], _TYPES[case["residual"]], _TYPES[case["branch"]]
        st = {"case": case, "residual": stream(B, L, d).to(dr), "branch": stream(B, L, d).mul_(0.5).to(db), "weight": None,
              "post": None, "gate": None}
        if case["pre"]:
            st["weight"] = (1.0 + 0.1 * normal(d)).to(db)
        if case["post"]:
            st["post"] = (0.5 + 0.1 * normal(d)).to(db)
        if case["gate"] != "none":
            shape = {"channel": (d,), "text": (B, 1, d), "token": (B, L, d)}[case["gate"]]
            st["gate"] = (0.3 + 0.5 * normal(*shape)).to(db)
        if case["op"] == "join_backward":  # what the forward returned, and the gradients that come back
            st["h"] = _plain_join(st)[0]
            st["residual"] = None
            st["dh"] = (1e-3 * normal(B, L, d)).to(dr)
            st["dy"] = (1e-3 * normal(B, L, d)).to(db) if case["pre"] else None
        return st
    dt = _TYPES[case["dtype"]]
    grads = [(1e-3 * torch.exp(normal(1)) * normal(*s)).to(dt) for s in _shapes(case)]
    st = {"case": case, "grads": grads, "out": None}
    if case["op"] == "clip":
        n = sum(x.numel() for x in grads)
        # gradients of these scales have a norm of 1e-3 to 1e-2 times the root of their number
        st["max_norm"] = math.sqrt(n) if case["within"] else 1e-4 * math.sqrt(n)
        if case["out"] != "none":
            st["out"] = [torch.zeros_like(x, dtype=_TYPES[case["out"]]) for x in grads]
    return st


# ---------------------------------------------------------------------------------------------------------- plain forms

def _plain_norm(x, weight, offset):
    x = x.float()
    return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * (offset + weight.float())


def _plain_norm_gradient(dy, x, weight, offset):
    """(dx, dweight) in fp32."""
    dy, x = dy.float(), x.float()
    r = 1.0 / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
    unit = x * r
    t = dy * (offset + weight.float())
    return (t - unit * (t * unit).mean(-1, keepdim=True)) * r, (dy * unit).flatten(0, -2).sum(0)


def _plain_join(st):
    case = st["case"]
    p = st["branch"].float() if st["post"] is None else _plain_norm(st["branch"], st["post"], 0.0)
    if st["gate"] is not None:
        p = p * st["gate"].float()
    h = st["residual"].float() + case["scale"] * p
    y = () if st["weight"] is None else (_plain_norm(h, st["weight"], 0.0).to(st["branch"].dtype),)
    return (h.to(st["residual"].dtype), *y)


def _plain_join_backward(st):
    case, post, gate = st["case"], st["post"], st["gate"]
    g = st["dh"].float()
    outs = {}
    if st["weight"] is not None:
        dn, dw = _plain_norm_gradient(st["dy"], st["h"], st["weight"], 0.0)
        g = g + dn
        outs["weight"] = dw.to(st["weight"].dtype)
    outs["residual"] = g.to(st["h"].dtype)
    t = g * case["scale"]
    if gate is not None:
        p = st["branch"].float() if post is None else _plain_norm(st["branch"], post, 0.0)
        dg = t * p
        if case["gate"] != "token":
            dg = dg.sum((0, 1)) if case["gate"] == "channel" else dg.sum(1, keepdim=True)
        outs["gate"] = dg.to(gate.dtype)
        t = t * gate.float()
    if post is not None:
        t, du = _plain_norm_gradient(t, st["branch"], post, 0.0)
        outs["post"] = du.to(post.dtype)
    outs["branch"] = t.to(st["branch"].dtype)
    return outs


def _plain_global_norm(grads):
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for x in grads:
        total = total + x.float().square().sum(dtype=torch.float64)
    return total.sqrt()


def _plain_clip(st):
    norm = _plain_global_norm(st["grads"])
    factor = (st["max_norm"] / (norm + CLIP_EPS)).clamp(max=1.0).float()
    out = st["grads"] if st["out"] is None else st["out"]
    for x, y in zip(st["grads"], out):
        y.copy_(x.float() * factor)
    return [norm.float(), *out]


def _plain(st):
    case = st["case"]
    op = case["op"]
    if op == "norm":
        return _plain_norm(st["x"], st["weight"], case["offset"]).to(st["x"].dtype)
    if op == "norm_backward":
        dx, dw = _plain_norm_gradient(st["dy"], st["x"], st["weight"], case["offset"])
        return dx.to(st["x"].dtype), dw.to(st["weight"].dtype)
    if op == "join":
        return _plain_join(st)
    if op == "join_backward":
        return _plain_join_backward(st)
    if op == "global_norm":
        return _plain_global_norm(st["grads"]).float()
    return _plain_clip(st)


# ------------------------------------------------------------------------------------------------------------- measured

def run(state):
    if not own:
        return _plain(state)
    case = state["case"]
    op = case["op"]
    if op.startswith("norm"):
        from lookatmyquant_b200 import norms
        if op == "norm":
            return norms.norm_forward(state["x"], state["weight"], eps=EPS, offset=case["offset"])
        return norms.norm_backward(state["dy"], state["x"], state["weight"], eps=EPS, offset=case["offset"])
    if op == "join":
        from lookatmyquant_b200 import norms
        h, y = norms.join_forward(state["residual"], state["branch"], state["weight"], post_weight=state["post"],
                                  gate=state["gate"], scale=case["scale"], eps=EPS)
        return (h,) if y is None else (h, y)
    if op == "join_backward":
        from lookatmyquant_b200 import norms
        grads = norms.join_backward(state["dh"], state["dy"], state["h"], state["branch"], state["weight"],
                                    post_weight=state["post"], gate=state["gate"], scale=case["scale"], eps=EPS)
        outs = dict(zip(("residual", "branch", "weight", "post", "gate"), grads))
        return {k: outs[k] for k in ("weight", "residual", "gate", "post", "branch") if outs[k] is not None}
    from lookatmyquant_b200 import gradients
    if op == "global_norm":
        return gradients.global_norm(state["grads"])
    norm = gradients.clip(state["grads"], state["max_norm"], out=state["out"])
    return [norm, *(state["grads"] if state["out"] is None else state["out"])]


_SIZES = {"bf16": 2, "fp32": 4}


def work(case):
    op = case["op"]
    if op.startswith("norm"):
        n, w = case["B"] * case["L"] * case["H"] * case["d"], case["d"]
        size = _SIZES[case["dtype"]]
        if op == "norm":
            return {"bytes": (2 * n + w) * size, "flops": 4 * n}
        return {"bytes": (3 * n + 2 * w) * size, "flops": 11 * n}
    if op.startswith("join"):
        n, d, r, b = case["B"] * case["L"] * case["d"], case["d"], _SIZES[case["residual"]], _SIZES[case["branch"]]
        gate = b * {"none": 0, "channel": d, "text": case["B"] * d, "token": n}[case["gate"]]
        weights = b * d * (case["pre"] + case["post"])
        if op == "join":
            return {"bytes": n * (2 * r + b + b * case["pre"]) + weights + gate,
                    "flops": n * (2 + 4 * case["pre"] + 4 * case["post"])}
        needs_branch = case["post"] or case["gate"] != "none"
        # without a post norm, a gate, a scale and a change of type, the branch's gradient is the residual's
        writes_branch = needs_branch or case["scale"] != 1.0 or r != b
        return {"bytes": n * (2 * r + case["pre"] * (r + b) + b * needs_branch + b * writes_branch) + 2 * (weights + gate),
                "flops": n * (2 + 11 * case["pre"] + 11 * case["post"] + 3 * (case["gate"] != "none"))}
    n = sum(math.prod(s) for s in _shapes(case))
    if op == "global_norm":
        return {"bytes": n * _SIZES[case["dtype"]], "flops": 2 * n}
    # within the bound nothing has to be written in place
    write = 0 if case["out"] == "none" and case["within"] else _SIZES[case["dtype" if case["out"] == "none" else "out"]]
    return {"bytes": n * (_SIZES[case["dtype"]] + write), "flops": (2 + (write > 0)) * n}


# --------------------------------------------------------------------------------------------------------------- 64 bits

def _unit(x):
    """Rows of mean square 1 (up to EPS), in 64 bits."""
    return x * torch.rsqrt(torch.einsum("...i,...i->...", x, x) / x.shape[-1] + EPS)[..., None]


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op.startswith("norm"):
        x = st["x"].double().requires_grad_(op == "norm_backward")
        w = st["weight"].double().requires_grad_(op == "norm_backward")
        y = _unit(x) * (w + case["offset"])
        return y if op == "norm" else torch.autograd.grad(y, (x, w), st["dy"].double())
    if op.startswith("join"):
        back = op == "join_backward"
        leaf = {k: None if st[k] is None else st[k].double().requires_grad_(back) for k in ("branch", "weight", "post", "gate")}
        p = leaf["branch"] if leaf["post"] is None else _unit(leaf["branch"]) * leaf["post"]
        q = case["scale"] * (p if leaf["gate"] is None else p * leaf["gate"])
        if not back:
            h = q + st["residual"].double()
            return (h,) if leaf["weight"] is None else (h, _unit(h) * leaf["weight"])
        outs, g = {}, st["dh"].double()
        if leaf["weight"] is not None:
            h = st["h"].double().requires_grad_(True)
            dn, outs["weight"] = torch.autograd.grad(_unit(h) * leaf["weight"], (h, leaf["weight"]), st["dy"].double())
            g = g + dn
        outs["residual"] = g
        names = [k for k in ("gate", "post", "branch") if leaf[k] is not None]
        outs.update(zip(names, torch.autograd.grad(q, [leaf[k] for k in names], g)))
        return outs
    norm = math.sqrt(sum(float(torch.linalg.vector_norm(x, dtype=torch.float64)) ** 2 for x in st["grads"]))
    first = torch.tensor(norm, dtype=torch.float64, device="cuda")
    if op == "global_norm":
        return first
    factor = min(1.0, st["max_norm"] / (norm + CLIP_EPS))
    return [first, *(x.double() * factor for x in st["grads"])]
