"""The training operators' measured cases: attention forwards and backwards, the scaled embedding lookup and its
gradient, and the Newton-Schulz orthogonalisation of an update.

`listed()` gives the cases, `draw(rng)` one more of the same ranges, `prepare(case, seed)` the tensors that a training
loop holds before the call, `run(state)` one call (`own` false: elementary fp32 torch operations; true: the package's
operators), `work(case)` the bytes and operations that the call cannot do without, and `exact(case, seed)` its result
in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5


# ---------------------------------------------------------------------------------------------------------------- cases

def _attention(op, B, Hq, Hkv, D, Lq, Lk, causal=True, pad="none"):
    return {"op": op, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "Lq": Lq, "Lk": Lk, "causal": causal, "pad": pad}


def listed():
    cases = [
        # one short text of odd length through a 15/5-head model (the smallest call a loop makes: latency)
        ("attention forward 77 tokens", _attention("attention_forward", 1, 15, 5, 64, 77, 77)),
        # held-out windows of the KL probe: 8 x 2048 tokens, 15/5 heads of 64
        ("attention forward windows", _attention("attention_forward", 8, 15, 5, 64, 2048, 2048)),
        # the gradient of one short text: row importance over single calibration texts
        ("attention backward 77 tokens", _attention("attention_backward", 1, 15, 5, 64, 77, 77)),
        # ragged texts padded on the left into one batch (one of them empty), 32/8 heads of 128, odd length
        ("attention backward ragged", _attention("attention_backward", 5, 32, 8, 128, 1337, 1337, True, "left")),
        # a fine-tuning step's long windows, 32/8 heads of 128
        ("attention backward 2 x 4096", _attention("attention_backward", 2, 32, 8, 128, 4096, 4096)),
        # one window's tokens looked up in a 49152 x 960 bf16 table
        ("lookup one window", {"op": "lookup", "V": 49152, "d": 960, "N": 2048, "dtype": "bf16", "pad": False}),
        # a large batch from a wide fp32 master table, padding tokens among them
        ("lookup batch", {"op": "lookup", "V": 131072, "d": 2560, "N": 32768, "dtype": "fp32", "pad": True}),
        # the table's gradient for one window: few tokens, most rows untouched
        ("lookup gradient one window", {"op": "lookup_gradient", "V": 49152, "d": 960, "N": 2048, "dtype": "fp32",
                                        "pad": False}),
        # the table's gradient for a large batch in bf16, with padding tokens and frequent tokens in long runs
        ("lookup gradient batch", {"op": "lookup_gradient", "V": 131072, "d": 2560, "N": 65536, "dtype": "bf16",
                                   "pad": True}),
        # one k_proj update of the 960-wide model (latency of the whole chain of products)
        ("newton-schulz 320 x 960", {"op": "newton_schulz", "batch": 1, "m": 320, "n": 960, "dtype": "fp32"}),
        # the four down_proj updates of a group of layers at once
        ("newton-schulz 4 x 960 x 2560", {"op": "newton_schulz", "batch": 4, "m": 960, "n": 2560, "dtype": "bf16"}),
        # one gate_proj update of the 2560-wide model
        ("newton-schulz 9728 x 2560", {"op": "newton_schulz", "batch": 1, "m": 9728, "n": 2560, "dtype": "fp32"}),
    ]
    return [dict(case, name=name) for name, case in cases]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attention_forward", "attention_backward", "attention_backward", "lookup", "lookup_gradient",
                     "lookup_gradient", "newton_schulz", "newton_schulz"])
    if op.startswith("attention"):
        Hq, Hkv, D = rng.choice([(15, 5, 64), (32, 8, 128), (32, 8, 128), (6, 6, 80), (8, 1, 96), (12, 4, 40)])
        B = _log_int(rng, 1, 8)
        most = min(4096, math.isqrt(2 * 32 * 4096 * 4096 * 128 // (B * Hq * D)))
        # over a single key the gradients of q and k are zero identically: nothing to measure
        Lk = _log_int(rng, 2 if op == "attention_backward" else 1, most)
        Lq = Lk if rng.random() < 0.7 else _log_int(rng, 1, Lk)
        return _attention(op, B, Hq, Hkv, D, Lq, Lk, rng.random() < 0.75, rng.choice(["none", "none", "left", "right"]))
    if op.startswith("lookup"):
        return {"op": op, "V": _log_int(rng, 256, 131072), "d": rng.choice([64, 320, 960, 1000, 1024, 2560]),
                "N": _log_int(rng, 1, 65536 if op == "lookup_gradient" else 32768),
                "dtype": rng.choice(["bf16", "fp32"]), "pad": rng.random() < 0.5}
    m, n = _log_int(rng, 16, 9728), _log_int(rng, 16, 9728)
    while min(m, n) ** 2 * (3 * max(m, n) + min(m, n)) > 2560 ** 2 * (3 * 9728 + 2560):
        m, n = (m + 1) // 2, (n + 1) // 2
    batch = rng.choice([1, 1, 2, 5]) if m * n < 2 ** 21 else 1
    return {"op": op, "batch": batch, "m": m, "n": n, "dtype": rng.choice(["fp32", "bf16"])}


# --------------------------------------------------------------------------------------------------------------- inputs

def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _key_ranges(case):
    """The keys [start, end) of each text of a padded batch: lengths from the whole window down to none."""
    B, Lk = case["B"], case["Lk"]
    lens = [Lk if B == 1 else round(Lk * (1.0 - b / (B - 1)) ** 0.5) for b in range(B)]
    if case["pad"] == "left":
        return [(Lk - n, Lk) for n in lens]
    if case["pad"] == "right":
        return [(0, n) for n in lens]
    return [(0, Lk)] * B


def _zipf(N, V, g):
    w = torch.arange(1, V + 1, dtype=torch.float64, device="cuda").pow(-1.1)
    u = torch.rand(N, dtype=torch.float64, device="cuda", generator=g) * w.sum()
    return torch.searchsorted(w.cumsum(0), u).clamp_(max=V - 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"].startswith("attention"):
        B, Hq, Hkv, D, Lq, Lk = (case[k] for k in ("B", "Hq", "Hkv", "D", "Lq", "Lk"))

        def heads(H, L, spread=1.0):  # (B, H, L, D) views of a projection's (B, L, H * D) output
            x = normal(B, L, H, D) * torch.exp(spread * 0.3 * normal(1, 1, H, D))
            return x.bfloat16().transpose(1, 2)
        st = {"case": case, "q": heads(Hq, Lq), "k": heads(Hkv, Lk), "v": heads(Hkv, Lk), "start": None, "end": None}
        if case["pad"] != "none":
            r = torch.tensor(_key_ranges(case), dtype=torch.int32, device="cuda")
            st["start"], st["end"] = r[:, 0].contiguous(), r[:, 1].contiguous()
        if case["op"] == "attention_backward":  # what the forward kept, and the gradient that comes back
            st["o"], st["lse"] = _plain_forward(st)
            st["do"] = heads(Hq, Lq) * 1e-3
        return st
    if case["op"].startswith("lookup"):
        V, d, N, dt = case["V"], case["d"], case["N"], _dtype(case)
        # frequent tokens anywhere in the table
        ids = torch.randperm(V, device="cuda", generator=g)[_zipf(N, V, g)]
        st = {"case": case, "ids": ids, "scale": math.sqrt(d), "padding": None}
        if case["pad"]:
            st["padding"] = 0
            ids[torch.rand(N, device="cuda", generator=g) < 0.1] = 0
        if case["op"] == "lookup":
            st["table"] = (0.02 * normal(V, d)).to(dt)
        else:
            st["dy"] = (1e-3 * normal(N, d)).to(dt)
        return st
    # a momentum: a few strong directions over noise, rows of differing scale
    b, m, n = case["batch"], case["m"], case["n"]
    r = max(1, min(m, n) // 16)
    G = normal(b, m, r) @ (normal(b, r, n) * torch.linspace(1.0, 0.1, r, device="cuda")[:, None]) / math.sqrt(r)
    G = (G + normal(b, m, n)) * torch.exp(0.5 * normal(b, m, 1)) * 1e-3
    return {"case": case, "G": (G if b > 1 else G[0]).to(_dtype(case))}


# ---------------------------------------------------------------------------------------------------------- plain forms

def _allowed(st):
    """(B, 1, 1, Lq, Lk): which keys each query sees."""
    Lq, Lk = st["q"].shape[2], st["k"].shape[2]
    j = torch.arange(Lk, device="cuda")
    ok = torch.ones(1, 1, 1, Lq, Lk, dtype=torch.bool, device="cuda")
    if st["case"]["causal"]:
        ok = ok & (j <= torch.arange(Lq, device="cuda")[:, None] + Lk - Lq)
    if st["start"] is not None:
        inside = (j >= st["start"][:, None]) & (j < st["end"][:, None])
        ok = ok & inside[:, None, None, None, :]
    return ok


def _grouped(st):
    """q, k, v in fp32 as (B, Hkv, group, L, D); k and v with one head per group."""
    B, Hq, Lq, D = st["q"].shape
    Hkv = st["k"].shape[1]
    return (st["q"].float().reshape(B, Hkv, Hq // Hkv, Lq, D), st["k"].float()[:, :, None], st["v"].float()[:, :, None])


def _plain_forward(st):
    q, k, v = _grouped(st)
    ok = _allowed(st)
    S = (q @ k.transpose(-1, -2) * q.shape[-1] ** -0.5).masked_fill_(~ok, -math.inf)
    top = S.amax(-1, keepdim=True)
    P = (S - top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = P.sum(-1, keepdim=True)
    o = (P @ v) / total.masked_fill(total == 0, 1.0)
    lse = (top + total.log())[..., 0]
    return o.reshape(st["q"].shape).bfloat16(), lse.reshape(st["q"].shape[:3])


def _plain_backward(st):
    q, k, v = _grouped(st)
    do = st["do"].float().reshape(q.shape)
    D = (do * st["o"].float().reshape(q.shape)).sum(-1, keepdim=True)
    scale = q.shape[-1] ** -0.5
    lse = st["lse"].reshape(*q.shape[:-1], 1)
    P = (q @ k.transpose(-1, -2) * scale - lse).exp_().masked_fill_(~_allowed(st), 0.0)
    dv = (P.transpose(-1, -2) @ do).sum(2)
    dS = P * (do @ v.transpose(-1, -2) - D)
    dq = (dS @ k) * scale
    dk = (dS.transpose(-1, -2) @ q).sum(2) * scale
    return dq.reshape(st["q"].shape).bfloat16(), dk.bfloat16(), dv.bfloat16()


def _plain_newton_schulz(G):
    X = G.float()
    tall = X.shape[-2] > X.shape[-1]
    X = X.transpose(-1, -2) if tall else X
    X = X / (X.square().sum((-2, -1), keepdim=True).sqrt() + 1e-7)
    a, b, c = NS_COEFFICIENTS
    for _ in range(NS_STEPS):
        A = X @ X.transpose(-1, -2)
        X = a * X + (b * A + c * (A @ A)) @ X
    return (X.transpose(-1, -2) if tall else X).bfloat16().contiguous()


def _plain(st):
    case = st["case"]
    if case["op"] == "attention_forward":
        return _plain_forward(st)
    if case["op"] == "attention_backward":
        return _plain_backward(st)
    if case["op"] == "newton_schulz":
        return _plain_newton_schulz(st["G"])
    live = None if st["padding"] is None else (st["ids"] != st["padding"])[:, None]
    if case["op"] == "lookup":
        y = st["table"][st["ids"]].float() * st["scale"]
        return (y if live is None else y * live).to(st["table"].dtype)
    dy = st["dy"].float() * st["scale"]
    dE = torch.zeros(case["V"], case["d"], device="cuda").index_add_(0, st["ids"], dy if live is None else dy * live)
    return dE.to(st["dy"].dtype)


# ------------------------------------------------------------------------------------------------------------- measured

def run(state):
    if not own:
        return _plain(state)
    case = state["case"]
    if case["op"].startswith("lookup"):
        from lookatmyquant_b200 import embedding
        if case["op"] == "lookup":
            return embedding.lookup(state["table"], state["ids"], scale=state["scale"], padding_idx=state["padding"])
        return embedding.lookup_gradient(state["dy"], state["ids"], case["V"], scale=state["scale"],
                                         padding_idx=state["padding"])
    if case["op"] == "newton_schulz":
        from lookatmyquant_b200 import orthogonal
        return orthogonal.newton_schulz(state["G"], steps=NS_STEPS, coefficients=NS_COEFFICIENTS)
    from lookatmyquant_b200 import attention
    if case["op"] == "attention_forward":
        return attention.forward(state["q"], state["k"], state["v"], causal=case["causal"], key_start=state["start"],
                                 key_end=state["end"])
    return attention.backward(state["do"], state["q"], state["k"], state["v"], state["o"], state["lse"],
                              causal=case["causal"], key_start=state["start"], key_end=state["end"])


def work(case):
    if case["op"].startswith("attention"):
        B, Hq, Hkv, D, Lq, Lk = (case[k] for k in ("B", "Hq", "Hkv", "D", "Lq", "Lk"))
        pairs = 0
        for lo, hi in _key_ranges(case):
            for i in range(Lq):
                end = min(hi, i + Lk - Lq + 1) if case["causal"] else hi
                pairs += max(0, end - lo)
        q, kv, rows = B * Hq * Lq * D * 2, B * Hkv * Lk * D * 2, B * Hq * Lq * 4
        if case["op"] == "attention_forward":
            return {"bytes": 2 * q + 2 * kv + rows, "flops": 4 * D * Hq * pairs}
        return {"bytes": 4 * q + 4 * kv + rows, "flops": 10 * D * Hq * pairs}
    if case["op"].startswith("lookup"):
        size = 2 if case["dtype"] == "bf16" else 4
        N, V, row = case["N"], case["V"], case["d"] * size
        if case["op"] == "lookup":  # the distinct rows that N Zipf draws meet, expected
            h = sum(r ** -1.1 for r in range(1, V + 1))
            distinct = sum(-math.expm1(N * math.log1p(-min(0.999999, r ** -1.1 / h))) for r in range(1, V + 1))
            return {"bytes": distinct * row + N * (row + 8), "flops": N * case["d"]}
        return {"bytes": N * (row + 8) + V * row, "flops": 2 * N * case["d"]}
    b, m, n = case["batch"], min(case["m"], case["n"]), max(case["m"], case["n"])
    size = 2 if case["dtype"] == "bf16" else 4
    flops = NS_STEPS * (m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n)
    return {"bytes": b * m * n * (size + 2), "flops": b * flops}


# --------------------------------------------------------------------------------------------------------------- 64 bits

def _exact_head(q, k, v, do, lo, hi, causal):
    """One head of one text in 64 bits: softmax over the keys [lo, hi), its gradients by the chain rule through the
    normalised weights (no lse)."""
    Lq, Lk, scale = q.shape[0], k.shape[0], 1.0 / math.sqrt(q.shape[1])
    o, lse = torch.zeros_like(q), torch.full((Lq,), -math.inf, dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    first = max(0, lo - (Lk - Lq)) if causal else 0  # the queries before see no key
    if hi <= lo or first >= Lq:
        return o, lse, dq, dk, dv
    z = torch.einsum("id,jd->ij", q[first:], k[lo:hi]) * scale
    if causal:
        i = torch.arange(first, Lq, device="cuda")[:, None]
        z[torch.arange(lo, hi, device="cuda")[None] > i + (Lk - Lq)] = -math.inf
    lse[first:] = torch.logsumexp(z, 1)
    p = torch.softmax(z, 1)
    o[first:] = p @ v[lo:hi]
    if do is not None:
        dv[lo:hi] = torch.einsum("ij,id->jd", p, do[first:])
        dp = torch.einsum("id,jd->ij", do[first:], v[lo:hi])
        dz = p * (dp - torch.einsum("ij,ij->i", p, dp)[:, None]) * scale
        dq[first:] = dz @ k[lo:hi]
        dk[lo:hi] = torch.einsum("ij,id->jd", dz, q[first:])
    return o, lse, dq, dk, dv


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"].startswith("attention"):
        q, k, v = (st[x].double() for x in "qkv")
        back = case["op"] == "attention_backward"
        do = st["do"].double() if back else None
        O, L = torch.empty_like(q), torch.empty(q.shape[:3], dtype=torch.float64, device="cuda")
        dQ, dK, dV = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
        group = q.shape[1] // k.shape[1]
        for b, (lo, hi) in enumerate(_key_ranges(case)):
            for h in range(q.shape[1]):
                e = h // group
                O[b, h], L[b, h], dQ[b, h], dk, dv = _exact_head(q[b, h], k[b, e], v[b, e], do[b, h] if back else None,
                                                                lo, hi, case["causal"])
                dK[b, e] += dk
                dV[b, e] += dv
        return (dQ, dK, dV) if back else (O, L)
    if case["op"].startswith("lookup"):
        scale, pad = st["scale"], st["padding"]
        if case["op"] == "lookup":
            y = torch.nn.functional.embedding(st["ids"], st["table"].double()) * scale
            if pad is not None:
                y[st["ids"] == pad] = 0.0
            return y
        dE = torch.zeros(case["V"], case["d"], dtype=torch.float64, device="cuda")
        dE.index_put_((st["ids"],), st["dy"].double(), accumulate=True)
        if pad is not None:
            dE[pad] = 0.0
        return dE * scale
    a, b, c = NS_COEFFICIENTS
    X = st["G"].double()
    X = X / (torch.linalg.matrix_norm(X, keepdim=True) + 1e-7)
    small = X.shape[-1] if X.shape[-2] > X.shape[-1] else X.shape[-2]
    eye = torch.eye(small, dtype=torch.float64, device="cuda")
    for _ in range(NS_STEPS):  # the polynomial of the Gram matrix, by Horner's rule, on the smaller side
        if X.shape[-2] > X.shape[-1]:
            gram = X.mT @ X
            X = X @ (a * eye + gram @ (b * eye + c * gram))
        else:
            gram = X @ X.mT
            X = (a * eye + gram @ (b * eye + c * gram)) @ X
    return X
