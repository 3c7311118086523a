"""LayerNorm and linear layers with an activation, forward and backward, as measurable cases.

``run`` makes the calls of ``basedxl_b200.ops`` where ``own`` is true, and evaluates the same formulas with elementary
PyTorch operations in fp32 where it is not.  ``listed()`` holds representative sizes, ``draw()`` more of the same ranges.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
ACTIVATIONS = ["none", "relu", "silu", "gelu", "gelu_tanh", "quick_gelu"]
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# The most that a drawn case may cost: what the largest listed ones do.
MAX_NORM_VALUES = 65536 * 1280
MAX_LINEAR_FLOPS = 2.0 * 8192 * 2560 * 10240
MAX_BACKWARD_FLOPS = 4.0 * 8192 * 1280 * 5120


def listed():
    return [
        # One pooled text embedding: the smallest call, bound by latency.
        {"name": "norm 1x1280", "kind": "norm", "rows": 1, "c": 1280, "dtype": "f16", "params": "same", "stats": False},
        # Training on a batch of activations whose width is no multiple of anything.
        {"name": "norm 4099x1285 f32", "kind": "norm", "rows": 4099, "c": 1285, "dtype": "f32", "params": "same", "stats": True},
        # A batch of sixteen 64x64 token maps with the widest blocks' channels: more than any cache holds.
        {"name": "norm 65536x1280", "kind": "norm", "rows": 65536, "c": 1280, "dtype": "bf16", "params": "f32", "stats": True},
        # Two prompts of 77 text tokens.
        {"name": "norm grad 154x2048", "kind": "norm_grad", "rows": 154, "c": 2048, "dtype": "f16", "params": "same"},
        # The tokens of a 2048x2048 image with guidance at the first transformer level; weights in fp32, as mixed precision keeps them.
        {"name": "norm grad 32768x640", "kind": "norm_grad", "rows": 32768, "c": 640, "dtype": "bf16", "params": "f32"},
        # A wide hidden layer in fp32.
        {"name": "norm grad 8192x5120 f32", "kind": "norm_grad", "rows": 8192, "c": 5120, "dtype": "f32", "params": "same"},
        # First layer of the time embedding, two rows (guidance): reads its weight once.
        {"name": "linear 2x320x1280", "kind": "linear", "m": 2, "k": 320, "n": 1280, "dtype": "f16", "act": "silu", "bias": True, "residual": False, "pre": False},
        # Extents that are no multiple of anything, with the first text encoder's activation and a residual.
        {"name": "linear 1000x1003x1501", "kind": "linear", "m": 1000, "k": 1003, "n": 1501, "dtype": "bf16", "act": "quick_gelu", "bias": True, "residual": True, "pre": False},
        # Feed-forward projection of a training step: z is kept for the backward pass.
        {"name": "linear 8192x1280x5120", "kind": "linear", "m": 8192, "k": 1280, "n": 5120, "dtype": "bf16", "act": "gelu", "bias": True, "residual": False, "pre": True},
        # The largest: bound by the tensor cores.
        {"name": "linear 8192x2560x10240", "kind": "linear", "m": 8192, "k": 2560, "n": 10240, "dtype": "f16", "act": "gelu_tanh", "bias": True, "residual": False, "pre": False},
        # Backward of a projection of the text tokens.
        {"name": "linear grad 154x1280x2048", "kind": "linear_grad", "m": 154, "k": 1280, "n": 2048, "dtype": "f16", "act": "gelu", "bias": True},
        # Backward of the feed-forward projection of a training step.
        {"name": "linear grad 8192x1280x5120", "kind": "linear_grad", "m": 8192, "k": 1280, "n": 5120, "dtype": "bf16", "act": "gelu", "bias": True},
    ]


def _log_int(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _extent(rng, lo, hi):
    """As often a multiple of 64, of 8 and any number."""
    n = _log_int(rng, lo, hi)
    of = rng.choice([1, 8, 64])
    return max(lo, n // of * of)


def draw(rng):
    while True:
        case = _draw(rng)
        if case["kind"] in ("norm", "norm_grad"):
            if case["rows"] * case["c"] <= MAX_NORM_VALUES // (2 if case["dtype"] == "f32" else 1):
                return case
        elif work(case)["flops"] <= (MAX_LINEAR_FLOPS if case["kind"] == "linear" else MAX_BACKWARD_FLOPS):
            return case


def _draw(rng):
    kind = rng.choice(["norm", "norm_grad", "linear", "linear_grad"])
    if kind in ("norm", "norm_grad"):
        case = {"kind": kind, "rows": _log_int(rng, 1, 65536), "c": _extent(rng, 16, 16384), "dtype": rng.choice(["f16", "bf16", "f32"]),
                "params": rng.choice(["same", "f32"])}
        return {**case, "stats": rng.random() < 0.5} if kind == "norm" else case
    case = {"kind": kind, "m": _log_int(rng, 1, 16384), "k": _extent(rng, 16, 5120), "n": _extent(rng, 16, 10240), "dtype": rng.choice(["f16", "bf16"]),
            "act": rng.choice(ACTIVATIONS), "bias": rng.random() < 0.75}
    return {**case, "residual": rng.random() < 0.5, "pre": rng.random() < 0.5} if kind == "linear" else case


def _normal(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *shape, scale=1.0, shift=0.0: torch.randn(*shape, device="cuda", generator=g) * scale + shift


def prepare(case, seed):
    rn, dt = _normal(seed), TYPES[case["dtype"]]
    if case["kind"] in ("norm", "norm_grad"):
        rows, c = case["rows"], case["c"]
        pt = dt if case["params"] == "same" else torch.float32
        # rows of a residual stream: each with a mean and a size of its own, channels of different sizes
        x = (rn(rows, c) * rn(c, scale=0.5).exp() * rn(rows, 1, scale=0.3).exp() + rn(rows, 1, scale=0.5)).to(dt)
        state = {"case": case, "x": x, "weight": rn(c, scale=0.2, shift=1.0).to(pt), "bias": rn(c, scale=0.2).to(pt)}
        if case["kind"] == "norm_grad":
            wide = x.double()
            state["dy"] = rn(rows, c).to(dt)
            state["mean"] = wide.mean(dim=-1).float()  # as the forward pass left them
            state["rstd"] = (wide.var(dim=-1, unbiased=False) + EPS).rsqrt().float()
        return state
    m, k, n = case["m"], case["k"], case["n"]
    state = {"case": case, "x": rn(m, k).to(dt), "weight": rn(n, k, scale=k**-0.5).to(dt)}
    if case["kind"] == "linear":
        state["bias"] = rn(n, scale=0.2).to(dt) if case["bias"] else None
        state["residual"] = rn(m, n).to(dt) if case["residual"] else None
    else:
        state["dy"] = rn(m, n).to(dt)
        # x W^T + b as the forward pass left it; without an activation none is kept
        state["pre"] = (state["x"].float() @ state["weight"].float().T + rn(n, scale=0.2)).to(dt) if case["act"] != "none" else None
    return state


def run(state):
    c = state["case"]
    if own:
        return _run_own(state, c)
    if c["kind"] == "norm":
        return _plain_norm(state, c)
    if c["kind"] == "norm_grad":
        return _plain_norm_grad(state)
    return _plain_linear(state, c) if c["kind"] == "linear" else _plain_linear_grad(state, c)


def _run_own(s, c):
    from basedxl_b200 import ops

    if c["kind"] == "norm":
        got = ops.layernorm_fwd(s["x"], s["weight"], s["bias"], EPS, want_stats=c["stats"])
        return dict(zip(("y", "mean", "rstd"), got)) if c["stats"] else {"y": got}
    if c["kind"] == "norm_grad":
        return dict(zip(("dx", "dweight", "dbias"), ops.layernorm_bwd(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])))
    if c["kind"] == "linear":
        got = ops.linear_act(s["x"], s["weight"], s["bias"], activation=c["act"], residual=s["residual"], want_pre=c["pre"])
        return dict(zip(("y", "pre"), got)) if c["pre"] else {"y": got}
    dx, dw, db = ops.linear_act_bwd(s["dy"], s["x"], s["weight"], s["pre"], activation=c["act"], want_dbias=c["bias"])
    return {"dx": dx, "dweight": dw, "dbias": db} if c["bias"] else {"dx": dx, "dweight": dw}


# ---- plain forms: fp32, rounded once at the end ----------------------------------------
def _plain_norm(s, c):
    x = s["x"].float()
    mean = x.mean(dim=-1, keepdim=True)
    d = x - mean
    rstd = ((d * d).mean(dim=-1, keepdim=True) + EPS).rsqrt()
    y = (d * rstd * s["weight"].float() + s["bias"].float()).to(s["x"].dtype)
    return {"y": y, "mean": mean[:, 0], "rstd": rstd[:, 0]} if c["stats"] else {"y": y}


def _plain_norm_grad(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    h = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy * s["weight"].float()
    dx = rstd * (g - g.mean(dim=-1, keepdim=True) - h * (g * h).mean(dim=-1, keepdim=True))
    pt = s["weight"].dtype
    return {"dx": dx.to(s["x"].dtype), "dweight": (dy * h).sum(dim=0).to(pt), "dbias": dy.sum(dim=0).to(pt)}


def _sigmoid(z):
    return 1.0 / (1.0 + torch.exp(-z))


def _tanh_argument(z):
    """gelu with tanh is z sigmoid(u) of this u."""
    return 2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)


def _plain_act(z, act):
    if act == "relu":
        return z * (z > 0)
    if act == "silu":
        return z * _sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return z * _sigmoid(_tanh_argument(z))
    return z * _sigmoid(1.702 * z) if act == "quick_gelu" else z


def _plain_act_grad(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        g = _sigmoid(_tanh_argument(z))
        return g + z * g * (1.0 - g) * 2.0 * math.sqrt(2.0 / math.pi) * (1.0 + 3 * 0.044715 * z * z)
    a = 1.702 if act == "quick_gelu" else 1.0
    g = _sigmoid(a * z)
    return g + a * z * g * (1.0 - g)


def _plain_linear(s, c):
    dt = s["x"].dtype
    z = s["x"].float() @ s["weight"].float().T
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _plain_act(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(dt), "pre": z.to(dt)} if c["pre"] else {"y": y.to(dt)}


def _plain_linear_grad(s, c):
    dt = s["x"].dtype
    dz = s["dy"].float()
    if c["act"] != "none":
        dz = dz * _plain_act_grad(s["pre"].float(), c["act"])
    out = {"dx": (dz @ s["weight"].float()).to(dt), "dweight": (dz.T @ s["x"].float()).to(dt)}
    return {**out, "dbias": dz.sum(dim=0).to(dt)} if c["bias"] else out


# ---- the same in 64 bits, from the definitions -------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    x, w = s["x"].double(), s["weight"].double()
    if case["kind"] in ("norm", "norm_grad"):
        b = s["bias"].double()
        leaves = [t.requires_grad_() for t in (x, w, b)]
        with torch.enable_grad():
            y = torch.nn.functional.layer_norm(x, (case["c"],), w, b, EPS)
        if case["kind"] == "norm_grad":
            return dict(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, leaves, s["dy"].double())))
        x = x.detach()
        var, mean = torch.var_mean(x, dim=-1, unbiased=False)
        return {"y": y.detach(), "mean": mean, "rstd": (var + EPS) ** -0.5} if case["stats"] else {"y": y.detach()}
    if case["kind"] == "linear":
        z = torch.nn.functional.linear(x, w, None if s["bias"] is None else s["bias"].double())
        y = _exact_act(z, case["act"])
        if s["residual"] is not None:
            y = y + s["residual"].double()
        return {"y": y, "pre": z} if case["pre"] else {"y": y}
    dz = s["dy"].double()
    if case["act"] != "none":
        z = s["pre"].double().requires_grad_()
        with torch.enable_grad():
            (dz,) = torch.autograd.grad(_exact_act(z, case["act"]), z, dz)
    out = {"dx": torch.einsum("mn,nk->mk", dz, w), "dweight": torch.einsum("mn,mk->nk", dz, x)}
    return {**out, "dbias": dz.sum(dim=0)} if case["bias"] else out


def _exact_act(z, act):
    f = torch.nn.functional
    if act == "quick_gelu":
        return z * torch.special.expit(1.702 * z)
    return {"none": lambda t: t, "relu": f.relu, "silu": f.silu, "gelu": f.gelu, "gelu_tanh": lambda t: f.gelu(t, approximate="tanh")}[act](z)


# ---- what a pass cannot do without ---------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] in ("norm", "norm_grad"):
        n, c = case["rows"] * case["c"], case["c"]
        params = 2.0 * c * (4 if case["params"] == "f32" else size)
        if case["kind"] == "norm":
            return {"bytes": 2.0 * size * n + params + 8.0 * case["rows"] * case["stats"], "flops": 8.0 * n}
        # the weight is read, the gradients of weight and bias are written
        return {"bytes": 3.0 * size * n + 1.5 * params + 8.0 * case["rows"], "flops": 16.0 * n}
    m, k, n = case["m"], case["k"], case["n"]
    if case["kind"] == "linear":
        return {"bytes": 2.0 * (m * k + n * k + n * case["bias"] + m * n * (1 + case["residual"] + case["pre"])), "flops": 2.0 * m * k * n}
    return {"bytes": 2.0 * (m * n * (1 + (case["act"] != "none")) + 2 * m * k + 2 * n * k + n * case["bias"]), "flops": 4.0 * m * k * n}
