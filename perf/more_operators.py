"""The operators of a block's MLP, measured as a user calls them.

  norm    layer norm or RMS norm of rows; in training with the gradients of the rows, the
          weight and the bias
  linear  activation(x W^T + bias) + residual as one product; in training with all gradients
  mlp     the branch as a whole, x + W2 activation(W1 norm(x) + b1) + b2; in training with all
          gradients

A case has ``rows`` tokens of ``width`` features. With ``own`` the calls are the package's,
else the same formulas in elementary operations in 32 bits. ``exact`` evaluates the
definitions in 64 bits. The activations are ``none``, ``relu2`` (the squared ReLU), ``gelu``
(by the normal distribution function) and ``silu``.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
EPS = {"layer": 1e-5, "rms": 1e-6}
ACTIVATIONS = ("none", "relu2", "gelu", "silu")


def listed():
    return [
        # The norm before the MLP of one sequence's decode step. Latency is all there is.
        dict(name="norm_one", kind="norm", dtype="bf16", norm="layer", rows=1, width=2048,
             train=False),
        # The synthetic copy model's step in training: 32 x 64 tokens of width 256.
        dict(name="norm_copy", kind="norm", dtype="fp32", norm="layer", rows=2048, width=256,
             train=True),
        # Ragged: a packed batch of an odd number of tokens, an odd width.
        dict(name="norm_odd", kind="norm", dtype="fp32", norm="rms", rows=30011, width=1001,
             train=True),
        # The wide single-layer model's training batch: 16 x 4096 tokens of width 4096.
        dict(name="norm_wide", kind="norm", dtype="bf16", norm="layer", rows=65536, width=4096,
             train=True),
        # One sequence's decode step: the first product of the streaming model's MLP.
        dict(name="linear_one", kind="linear", dtype="bf16", rows=1, width=2048, out=8192,
             activation="gelu", bias=True, residual=False, train=False),
        # A step of the streaming decode benchmark's batch of 256: the second product.
        dict(name="linear_batch", kind="linear", dtype="bf16", rows=256, width=8192, out=2048,
             activation="none", bias=True, residual=True, train=False),
        # Odd widths on both sides, in training, fp32 as the small models train.
        dict(name="linear_odd", kind="linear", dtype="fp32", rows=3001, width=1001, out=777,
             activation="silu", bias=True, residual=True, train=True),
        # The first product of a training step of the streaming model.
        dict(name="linear_train", kind="linear", dtype="bf16", rows=8192, width=2048, out=8192,
             activation="gelu", bias=True, residual=False, train=True),
        # The copy model's MLP in training.
        dict(name="mlp_copy", kind="mlp", dtype="fp32", norm="rms", rows=2048, width=256, inner=1024,
             activation="relu2", bias=False, train=True),
        # The streaming decode benchmark's MLP: 256 sequences, one token each.
        dict(name="mlp_decode", kind="mlp", dtype="bf16", norm="rms", rows=256, width=2048,
             inner=8192, activation="relu2", bias=False, train=False),
        # The streaming model's MLP in training: 16 x 4096 tokens.
        dict(name="mlp_wide", kind="mlp", dtype="bf16", norm="rms", rows=65536, width=2048,
             inner=8192, activation="relu2", bias=False, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "linear", "linear", "mlp"))
    dtype = rng.choice(("fp32", "bf16"))
    train = rng.random() < 0.6
    case = dict(kind=kind, dtype=dtype, train=train)
    if kind != "linear":
        case["norm"] = rng.choice(("layer", "rms"))
    if kind == "norm":
        width = _log(rng, 16, 8192)
        rows = _log(rng, 1, min(200000, 268_000_000 // width))
        case.update(rows=rows, width=width)
        return case
    # Multiply-adds of one product: fp32 products run at a tenth of bf16's rate.
    most = 1_000_000_000_000 if dtype == "bf16" else 60_000_000_000
    width, inner = _log(rng, 16, 8192), _log(rng, 16, 8192)
    rows = _log(rng, 1, min(65536, most // (width * inner)))
    case.update(rows=rows, width=width, bias=rng.random() < 0.5)
    if kind == "linear":
        case.update(out=inner, activation=rng.choice(ACTIVATIONS), residual=rng.random() < 0.5)
    else:
        case.update(inner=inner, activation=rng.choice(ACTIVATIONS[1:]))
    return case


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _stream_rows(g, rows, width):
    """Rows of a residual stream: sizes that differ by row, a mean, a few loud features."""
    x = _randn(g, rows, width)
    x.mul_(0.5 + torch.rand(rows, 1, generator=g, device=DEVICE) * 2).add_(0.2 * _randn(g, rows, 1))
    loud = torch.randint(0, width, (max(1, width // 200),), generator=g, device=DEVICE)
    x[:, loud] *= 6.0
    return x


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype, kind, n, width = TYPES[case["dtype"]], case["kind"], case["rows"], case["width"]
    t = {}
    if kind == "linear":
        t["x"] = _randn(g, n, width)
        t["weight"] = _randn(g, case["out"], width).mul_(1.0 / math.sqrt(width))
        if case["bias"]:
            t["bias"] = _randn(g, case["out"]).mul_(0.3)
        if case["residual"]:
            t["residual"] = _randn(g, n, case["out"])
    else:
        t["x"] = _stream_rows(g, n, width)
        t["norm_weight"] = 1.0 + 0.2 * _randn(g, width)
        if case["norm"] == "layer":
            t["norm_bias"] = 0.2 * _randn(g, width)
    if kind == "mlp":
        inner = case["inner"]
        t["w1"] = _randn(g, inner, width).mul_(1.0 / math.sqrt(width))
        t["w2"] = _randn(g, width, inner).mul_(1.0 / math.sqrt(inner))
        if case["bias"]:
            t["b1"], t["b2"] = 0.3 * _randn(g, inner), 0.3 * _randn(g, width)
    t = {k: v.to(dtype).requires_grad_(case["train"]) for k, v in t.items()}
    state = dict(case=case, t=t)
    if case["train"]:
        state["grad"] = _randn(g, n, case.get("out", width)).to(dtype)
    return state


# ---- the formulas in elementary operations, 32 bits ------------------------------------------
def _norm(x, weight, bias, eps):
    """(rows normed, their scale, the normed rows with weight and bias)."""
    if bias is not None:
        x = x - x.mean(dim=1, keepdim=True)
    scale = torch.rsqrt((x * x).mean(dim=1, keepdim=True) + eps)
    unit = x * scale
    return unit, scale, unit * weight if bias is None else unit * weight + bias


def _norm_grad(g, unit, scale, weight, center):
    gw = g * weight
    d = gw - unit * (gw * unit).mean(dim=1, keepdim=True)
    if center:
        d = d - gw.mean(dim=1, keepdim=True)
    return d * scale, (g * unit).sum(dim=0), g.sum(dim=0)


def _activated(z, name):
    """(activation, its derivative)."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu2":
        r = z.clamp(min=0)
        return r * r, 2 * r
    if name == "gelu":
        tail = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * tail, tail + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s))


def _plain(state):
    case, kind = state["case"], state["case"]["kind"]
    t = {k: v.detach().float() for k, v in state["t"].items()}
    g = state["grad"].float() if case["train"] else None
    out = {}
    if kind == "linear":
        z = t["x"] @ t["weight"].t()
        if case["bias"]:
            z = z + t["bias"]
        y, d = _activated(z, case["activation"])
        out["out"] = y + t["residual"] if case["residual"] else y
        if case["train"]:
            dz = g * d
            out.update(x=dz @ t["weight"], weight=dz.t() @ t["x"])
            if case["bias"]:
                out["bias"] = dz.sum(dim=0)
            if case["residual"]:
                out["residual"] = g
    else:
        center = case["norm"] == "layer"
        unit, scale, y = _norm(t["x"], t["norm_weight"], t.get("norm_bias"), EPS[case["norm"]])
        if kind == "norm":
            out["out"] = y
        else:
            z = y @ t["w1"].t()
            if case["bias"]:
                z = z + t["b1"]
            h, d = _activated(z, case["activation"])
            o = t["x"] + h @ t["w2"].t()
            out["out"] = o + t["b2"] if case["bias"] else o
        if case["train"]:
            gn = g
            if kind == "mlp":
                dz = (g @ t["w2"]) * d
                gn = dz @ t["w1"]
                out.update(w1=dz.t() @ y, w2=g.t() @ h)
                if case["bias"]:
                    out.update(b1=dz.sum(dim=0), b2=g.sum(dim=0))
            dx, dw, db = _norm_grad(gn, unit, scale, t["norm_weight"], center)
            out["x"] = dx if kind == "norm" else g + dx
            out["norm_weight"] = dw
            if center:
                out["norm_bias"] = db
    dtype = state["t"]["x"].dtype
    return {k: v.to(dtype) for k, v in out.items()}


# ---- the package's calls ---------------------------------------------------------------------
def _package(state):
    import dabsn_amd

    case, kind, t = state["case"], state["case"]["kind"], state["t"]
    if kind == "linear":
        out = dabsn_amd.fused_linear(t["x"], t["weight"], t.get("bias"),
                                     activation=case["activation"], residual=t.get("residual"))
    elif kind == "mlp":
        out = dabsn_amd.fused_mlp(t["x"], t["w1"], t["w2"], t.get("b1"), t.get("b2"),
                                  norm=case["norm"], norm_weight=t["norm_weight"],
                                  norm_bias=t.get("norm_bias"), eps=EPS[case["norm"]],
                                  activation=case["activation"])
    elif case["norm"] == "layer":
        out = dabsn_amd.layer_norm(t["x"], t["norm_weight"], t["norm_bias"], eps=EPS["layer"])
    else:
        out = dabsn_amd.rms_norm(t["x"], t["norm_weight"], eps=EPS["rms"])
    if not case["train"]:
        return {"out": out}
    grads = torch.autograd.grad(out, list(t.values()), state["grad"])
    return {"out": out, **dict(zip(t, grads))}


def run(state):
    return _package(state) if own else _plain(state)


def work(case):
    kind, size, n, k = case["kind"], 2 if case["dtype"] == "bf16" else 4, case["rows"], case["width"]
    passes = 3 if case["train"] else 1
    if kind == "norm":
        # Forward: rows in and out; backward: rows and their gradients in, gradients out.
        vectors = k * (2 if case["norm"] == "layer" else 1) * (2 if case["train"] else 1)
        return {"bytes": size * (n * k * (4 if case["train"] else 2) + vectors),
                "flops": n * k * (18 if case["train"] else 7)}
    if kind == "linear":
        f = case["out"]
        vectors = f if case["bias"] else 0
        rows = n * (k + f) + (n * f if case["residual"] else 0)
        if case["train"]:
            rows += n * (k + f) + f * k + vectors
        return {"bytes": size * (rows + f * k + vectors), "flops": passes * 2 * n * k * f}
    f = case["inner"]
    weights = 2 * f * k + k * (2 if case["norm"] == "layer" else 1) + (f + k if case["bias"] else 0)
    return {"bytes": size * (n * k * (4 if case["train"] else 2) + weights * (2 if case["train"] else 1)),
            "flops": passes * 4 * n * k * f}


# ---- the definitions in 64 bits --------------------------------------------------------------
def _exact_activation(z, name):
    if name == "none":
        return z, 1.0
    if name == "relu2":
        return torch.where(z > 0, z * z, 0.0), torch.where(z > 0, 2 * z, 0.0)
    if name == "gelu":
        below = torch.special.ndtr(z)
        return z * below, below + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    near = 1 / (1 + torch.exp(-z))
    return z * near, near + z * near / (1 + torch.exp(z))


def _exact_norm(x, case, weight, bias):
    """(normed rows, a function from their gradient to those of x, weight and bias)."""
    mean = x.mean(dim=1, keepdim=True) if case["norm"] == "layer" else 0.0
    var = ((x - mean) ** 2).sum(dim=1, keepdim=True) / x.shape[1]
    std = torch.sqrt(var + EPS[case["norm"]])
    unit = (x - mean) / std

    def back(g):
        u = g * weight
        along = (u * unit).sum(dim=1, keepdim=True) / x.shape[1]
        level = u.sum(dim=1, keepdim=True) / x.shape[1] if case["norm"] == "layer" else 0.0
        return (u - level - along * unit) / std, torch.sum(g * unit, 0), torch.sum(g, 0)

    return (unit * weight if bias is None else torch.addcmul(bias, unit, weight)), back


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    t = {k: v.detach().to(torch.float64) for k, v in state["t"].items()}
    g = state["grad"].to(torch.float64) if case["train"] else None
    if kind == "linear":
        z = torch.mm(t["x"], t["weight"].t())
        z += t["bias"] if case["bias"] else 0.0
        value, slope = _exact_activation(z, case["activation"])
        out = {"out": value + (t["residual"] if case["residual"] else 0.0)}
        if case["train"]:
            dz = g * slope
            out["x"] = torch.mm(dz, t["weight"])
            out["weight"] = torch.mm(dz.t(), t["x"])
            if case["bias"]:
                out["bias"] = torch.sum(dz, 0)
            if case["residual"]:
                out["residual"] = g
        return out
    y, back = _exact_norm(t["x"], case, t["norm_weight"], t.get("norm_bias"))
    if kind == "norm":
        out, upstream = {"out": y}, g
    else:
        z = torch.mm(y, t["w1"].t())
        z += t["b1"] if case["bias"] else 0.0
        h, slope = _exact_activation(z, case["activation"])
        total = torch.addmm(t["x"], h, t["w2"].t())
        out = {"out": total + (t["b2"] if case["bias"] else 0.0)}
        if case["train"]:
            dz = torch.mm(g, t["w2"]) * slope
            upstream = torch.mm(dz, t["w1"])
            out["w1"], out["w2"] = torch.mm(dz.t(), y), torch.mm(g.t(), h)
            if case["bias"]:
                out["b1"], out["b2"] = torch.sum(dz, 0), torch.sum(g, 0)
    if case["train"]:
        dx, dw, db = back(upstream)
        out["x"] = dx + g if kind == "mlp" else dx
        out["norm_weight"] = dw
        if case["norm"] == "layer":
            out["norm_bias"] = db
    return out
