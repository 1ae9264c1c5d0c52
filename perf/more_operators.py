"""The feed-forward half of a block in dense weights, timed: a gated feed-forward block and the norms around it, with their
gradients.

    G = x W1^T   U = x W3^T   M = act(G, U)   y = M W2^T

with W1, W3 ``[inter, hidden]`` and W2 ``[hidden, inter]``, and, between two blocks,

    z = post * y / rms(y)   h = scale * residual + gate * z   n = weight * h / rms(h)

Four kinds of case:

* ``ffn``        the block forward
* ``ffn_grad``   forward and backward: y and the gradients of x and the three weights
* ``norm``       h and n
* ``norm_grad``  both, and the gradients of residual, y, the norms' weights and the gate
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # The smallest block: one token through the tiny expert's shapes.
        {"name": "ffn_tiny", "kind": "ffn", "t": 1, "h": 256, "i": 512, "act": "swiglu", "dtype": "bf16"},
        # One generated token through a dense expert of the 7168 x 2048 layer: its weights are read once.
        {"name": "ffn_token", "kind": "ffn", "t": 1, "h": 7168, "i": 2048, "act": "swiglu", "dtype": "bf16"},
        # A decode batch, an odd number of rows.
        {"name": "ffn_batch", "kind": "ffn", "t": 45, "h": 5120, "i": 1536, "act": "situ", "dtype": "f16"},
        # A short prompt on a block whose channels fill no tile.
        {"name": "ffn_ragged", "kind": "ffn", "t": 333, "h": 2056, "i": 1400, "act": "swiglu", "dtype": "f16"},
        # A long prompt: the matrix cores' case.
        {"name": "ffn_prompt", "kind": "ffn", "t": 4096, "h": 7168, "i": 2048, "act": "swiglu", "dtype": "bf16"},
        # The gradients of the few rows that a calibration batch routes to an expert.
        {"name": "ffn_grad_rows", "kind": "ffn_grad", "t": 27, "h": 5120, "i": 1536, "act": "situ", "dtype": "bf16"},
        # A small training step.
        {"name": "ffn_grad_batch", "kind": "ffn_grad", "t": 500, "h": 5120, "i": 1536, "act": "swiglu", "dtype": "f16"},
        # The largest: a training step of 4096 rows.
        {"name": "ffn_grad_full", "kind": "ffn_grad", "t": 4096, "h": 7168, "i": 2048, "act": "swiglu", "dtype": "bf16"},
        # Between two blocks while one token is generated: latency alone.
        {"name": "norm_token", "kind": "norm", "t": 1, "h": 7168, "residual": "bf16", "post": True, "gate": "channel",
         "scale": 1.0, "params": "bf16", "dtype": "bf16"},
        # Between two blocks of a long prompt, the residual stream in 32 bits.
        {"name": "norm_prompt", "kind": "norm", "t": 4096, "h": 7168, "residual": "f32", "post": True, "gate": "channel",
         "scale": 0.5, "params": "f32", "dtype": "bf16"},
        # Gradients where every row has a gate of its own and the block no norm behind it.
        {"name": "norm_grad_ragged", "kind": "norm_grad", "t": 333, "h": 2056, "residual": "f16", "post": False,
         "gate": "row", "scale": 1.0, "params": "f32", "dtype": "f16"},
        # The same of a training step: both norms, a gate for each channel.
        {"name": "norm_grad_full", "kind": "norm_grad", "t": 8192, "h": 5120, "residual": "bf16", "post": True,
         "gate": "channel", "scale": 0.7, "params": "f32", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["ffn", "ffn", "ffn_grad", "ffn_grad", "norm", "norm_grad"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    h = 8 * _log(rng, 8, 896)
    if kind.startswith("ffn"):
        i = 8 * _log(rng, 8, 512)
        most = 4096 * 7168 * 2048 // (h * i)  # no more than the largest listed case
        return {"kind": kind, "t": _log(rng, 1, max(1, min(8192, most))), "h": h, "i": i,
                "act": rng.choice(["swiglu", "situ"]), "dtype": dtype}
    return {"kind": kind, "t": _log(rng, 1, 8192 * 5120 // max(h, 2560)), "h": h, "residual": rng.choice(["f32", dtype]),
            "post": rng.random() < 0.7, "gate": rng.choice(["none", "channel", "channel", "row"]),
            "scale": rng.choice([1.0, 0.5, 0.7]), "params": rng.choice(["f32", dtype]), "dtype": dtype}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed) + 1)
    dtype, kind, t, h = DTYPE[case["dtype"]], case["kind"], case["t"], case["h"]
    grad = kind.endswith("_grad")
    state = {"case": dict(case)}

    def normal(*shape, scale=1.0):
        return scale * torch.randn(shape, generator=gen, device=DEV)

    def strong(rows, channels):  # a few strong channels
        return normal(rows, channels) * (1 + 2 * torch.rand(channels, generator=gen, device=DEV) ** 8)

    if kind.startswith("ffn"):
        i = case["i"]
        state["x"] = strong(t, h).to(dtype)
        state["w1"] = normal(i, h, scale=h**-0.5).to(dtype)
        state["w3"] = normal(i, h, scale=h**-0.5).to(dtype)
        state["w2"] = normal(h, i, scale=i**-0.5).to(dtype)
        state["leaves"] = ["x", "w1", "w3", "w2"]
        if grad:
            state["dy"] = normal(t, h, scale=0.1).to(dtype)
    else:
        params = DTYPE[case["params"]]
        state["residual"] = (3 * strong(t, h)).to(DTYPE[case["residual"]])
        state["y"] = strong(t, h).to(dtype)
        state["weight"] = (1 + normal(h, scale=0.2)).to(params)
        state["post"] = (1 + normal(h, scale=0.2)).to(params) if case["post"] else None
        state["gate"] = None
        if case["gate"] == "channel":
            state["gate"] = (0.5 + normal(h, scale=0.2)).to(params)
        elif case["gate"] == "row":
            state["gate"] = torch.sigmoid(normal(t, 1)).to(params)
        state["leaves"] = [k for k in ("residual", "y", "weight", "post", "gate") if state[k] is not None]
        if grad:
            state["dh"] = normal(t, h, scale=0.1).to(DTYPE[case["residual"]])
            state["dn"] = normal(t, h, scale=0.1).to(dtype)
    if grad:
        for k in state["leaves"]:
            state[k].requires_grad_()
    return state


# ---------------------------------------------------------------------------
# The plain forms, and the framework's
# ---------------------------------------------------------------------------


def _activate(g, u, act):
    """The activation and its derivatives by gate and up."""

    s = torch.sigmoid(g)
    if act == "swiglu":
        return g * s * u, u * s * (1 + g * (1 - s)), g * s
    a, b = torch.tanh(g / 4), torch.tanh(u / 25)
    f = 4 * a * s
    return f * 25 * b, 25 * b * ((1 - a * a) * s + f * (1 - s)), f * (1 - b * b)


def _ffn(state, case):
    x, w1, w3, w2 = (state[k].float() for k in state["leaves"])
    m, by_g, by_u = _activate(x @ w1.T, x @ w3.T, case["act"])
    out = {"y": m @ w2.T}
    if case["kind"] == "ffn_grad":
        dy = state["dy"].float()
        dm = dy @ w2
        dg, du = dm * by_g, dm * by_u
        out |= {"x": dg @ w1 + du @ w3, "w1": dg.T @ x, "w3": du.T @ x, "w2": dy.T @ m}
    return {k: v.to(state["x"].dtype) for k, v in out.items()}


def _norm(state, case):
    f = {k: state[k].float() for k in state["leaves"]}
    y, weight = f["y"], f["weight"]
    post, gate = f.get("post"), f.get("gate")
    z = y
    if post is not None:
        sy = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
        yhat = y * sy
        z = yhat * post
    h = case["scale"] * f["residual"] + (z if gate is None else gate * z)
    sh = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    out = {"h": h.to(state["residual"].dtype), "n": (h * sh * weight).to(state["y"].dtype)}
    if case["kind"] == "norm":
        return out
    dn = state["dn"].float()
    dnw = dn * weight
    dh = state["dh"].float() + sh * (dnw - h * sh * sh * (dnw * h).mean(-1, keepdim=True))
    dz = dh if gate is None else gate * dh
    grads = {"residual": case["scale"] * dh, "y": dz, "weight": (dn * h * sh).sum(0)}
    if post is not None:
        grads["post"] = (dz * yhat).sum(0)
        d = dz * post
        grads["y"] = sy * (d - yhat * (d * yhat).mean(-1, keepdim=True))
    if gate is not None:
        grads["gate"] = (dh * z).sum(0) if gate.dim() == 1 else (dh * z).sum(-1, keepdim=True)
    return out | {"d" + k: grads[k].to(state[k].dtype) for k in state["leaves"]}


def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return _ffn(state, case) if case["kind"].startswith("ffn") else _norm(state, case)
    leaves = [state[k] for k in state["leaves"]]
    if case["kind"].startswith("ffn"):
        from qsrt_amd.gated_ffn import gated_ffn

        y = gated_ffn(*leaves, activation=case["act"])
        if case["kind"] == "ffn":
            return {"y": y}
        return {"y": y.detach()} | dict(zip(state["leaves"], torch.autograd.grad(y, leaves, state["dy"])))
    from qsrt_amd.block_norm import residual_norm

    h, n = residual_norm(state["residual"], state["y"], state["weight"], post_weight=state["post"], gate=state["gate"],
                         scale=case["scale"], eps=EPS)
    if case["kind"] == "norm":
        return {"h": h, "n": n}
    grads = torch.autograd.grad((h, n), leaves, (state["dh"], state["dn"]))
    return {"h": h.detach(), "n": n.detach()} | {"d" + k: g for k, g in zip(state["leaves"], grads)}


# ---------------------------------------------------------------------------
# In 64 bits, from the definition: gradients by differentiating it
# ---------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    grad = case["kind"].endswith("_grad")
    leaf = {k: state[k].detach().double().requires_grad_(grad) for k in state["leaves"]}
    if case["kind"].startswith("ffn"):
        g, u = (torch.nn.functional.linear(leaf["x"], leaf[w]) for w in ("w1", "w3"))
        if case["act"] == "swiglu":
            m = g / (1 + torch.exp(-g)) * u
        else:
            m = 100 * torch.tanh(0.25 * g) / (1 + torch.exp(-g)) * torch.tanh(0.04 * u)
        y = torch.nn.functional.linear(m, leaf["w2"])
        if not grad:
            return {"y": y}
        return {"y": y.detach()} | dict(zip(leaf, torch.autograd.grad(y, list(leaf.values()), state["dy"].double())))
    z = leaf["y"]
    if "post" in leaf:
        z = leaf["post"] * z / (z.square().mean(1) + EPS).sqrt()[:, None]
    h = leaf["residual"] * case["scale"] + z * leaf.get("gate", 1.0)
    n = leaf["weight"] * h / (h.square().mean(1) + EPS).sqrt()[:, None]
    if not grad:
        return {"h": h, "n": n}
    grads = torch.autograd.grad((h, n), list(leaf.values()), (state["dh"].double(), state["dn"].double()))
    return {"h": h.detach(), "n": n.detach()} | {"d" + k: g for k, g in zip(leaf, grads)}


def work(case):
    """Inputs and parameters once, outputs and gradients once; the products alone as operations of the block."""

    t, h, grad = case["t"], case["h"], case["kind"].endswith("_grad")
    if case["kind"].startswith("ffn"):
        i = case["i"]
        rows, weights = 2 * t * h, 2 * 3 * h * i
        return {"bytes": float((4 * rows + 2 * weights) if grad else (2 * rows + weights)),
                "flops": (18.0 if grad else 6.0) * t * h * i}
    size = {"f32": 4, "bf16": 2, "f16": 2}
    rows = t * h * (size[case["residual"]] + size[case["dtype"]])
    vectors = h * (1 + case["post"] + (case["gate"] == "channel")) + t * (case["gate"] == "row")
    passes = 4 if grad else 2  # in and out, and the same of the gradients
    return {"bytes": float(passes * rows + (2 if grad else 1) * vectors * size[case["params"]]),
            "flops": (30.0 if grad else 10.0) * t * h}
