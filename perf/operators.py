"""The cases at which the operators of sgnn_amd.functional and sgnn_amd.muon are measured.

  layer_norm      rows normalised, scaled and shifted (+ residual); with its backward pass, the
                  reductions of the weight's and the bias's gradient among it
  linear          act(x W^T + b) (+ residual), with its backward pass
  newton_schulz   matrices orthogonalised by five quintic Newton-Schulz steps (the Muon update)

A case is a dict of plain values.  `run` computes it from what `prepare` made: in plain torch
operations in 32 bits while `own` is false, by the framework's operators while it is true.
`exact` computes the same outputs in 64 bits.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
QUINTIC = (3.4445, -4.7750, 2.0315)
EPS = 1e-5
NORM_EPS = 1e-7


def _ln(name, rows, width, dtype, train, residual):
    return {"name": name, "op": "layer_norm", "rows": rows, "width": width, "dtype": dtype, "train": train,
            "residual": residual}


def _lin(name, rows, k, n, dtype, act, train, residual):
    return {"name": name, "op": "linear", "rows": rows, "in": k, "out": n, "dtype": dtype, "act": act, "train": train,
            "residual": residual}


def _ns(name, count, rows, cols, dtype):
    return {"name": name, "op": "newton_schulz", "count": count, "rows": rows, "cols": cols, "dtype": dtype}


def listed():
    return [
        # the node latents of the 80-particle scene in inference: one launch's latency
        _ln("ln_scene", 80, 64, "f32", False, True),
        # the message LayerNorm of a training step, one row per edge of a 20k-particle graph
        _ln("ln_edges_train", 200003, 128, "f32", True, False),
        # a wide 16-bit block's norm over a training batch of rows
        _ln("ln_wide_train", 16384, 4096, "bf16", True, False),
        # a width that is no multiple of a vector, residual form
        _ln("ln_odd_train", 5003, 771, "f16", True, True),
        # a decoder's hidden Linear on the 80-particle scene: one launch's latency
        _lin("lin_scene", 80, 64, 64, "f32", "relu", False, False),
        # one row through a wide layer: the weight's bytes are the work
        _lin("lin_row", 1, 4096, 4096, "bf16", "gelu_tanh", False, True),
        # the message MLP's first Linear in training: [x_i, x_j, e] rows of hidden 128
        _lin("lin_edges_train", 200003, 384, 128, "f32", "silu", True, False),
        # a wide block's expanding Linear over a training batch
        _lin("lin_wide_train", 8192, 2048, 8192, "bf16", "gelu", True, False),
        # odd in every dimension, residual form
        _lin("lin_odd_train", 1037, 515, 771, "f16", "silu", True, True),
        # one small weight: one launch's latency
        _ns("ns_small", 1, 64, 64, "f32"),
        # the first Linears of the ten edge MLPs of a hidden-128 simulator
        _ns("ns_blocks", 10, 128, 384, "f32"),
        # one wide layer's 16-bit update, taller than wide
        _ns("ns_wide", 1, 4096, 2048, "bf16"),
    ]


def _size(rng, low, high):
    """Log-uniform; half of the draws are multiples of 16 (where there are any), the others any number."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and v >= 16:
        v -= v % 16
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(("layer_norm", "linear", "newton_schulz"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    if op == "layer_norm":
        width = _size(rng, 16, 8192)
        rows = _size(rng, 1, min(262144, (1 << 26) // width))
        return {"op": op, "rows": rows, "width": width, "dtype": dtype, "train": rng.random() < 0.6,
                "residual": rng.random() < 0.4}
    if op == "linear":
        k, n = _size(rng, 16, 8192), _size(rng, 16, 8192)
        most = min(262144, (1 << 26) // max(k, n), (1 << 35) // (k * n))
        act, train = rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu")), rng.random() < 0.6
        # relu's slope jumps at 0: on which side a z of 1e-8 falls is beyond a 32-bit sum, and one row in the
        # wrong place is more than 32-bit gradients may be off, so these are drawn with the smooth ones
        act = "silu" if act == "relu" and train and dtype == "f32" else act
        return {"op": op, "rows": _size(rng, 1, most), "in": k, "out": n, "dtype": dtype, "act": act, "train": train,
                "residual": rng.random() < 0.4}
    rows, cols = _size(rng, 16, 3000), _size(rng, 16, 3000)
    count = _size(rng, 1, max(1, min(48, (1 << 33) // (min(rows, cols) * rows * cols))))
    return {"op": op, "count": count, "rows": rows, "cols": cols, "dtype": dtype}


def _given(case, seed):
    """The inputs, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] == "newton_schulz":
        # a mini-batch gradient: noise in every direction and a few strong ones
        b, m, n = case["count"], case["rows"], case["cols"]
        strong = normal(b, m, 4) @ normal(b, 4, n).contiguous()
        return {"g": (0.02 * normal(b, m, n) + 0.02 * strong).to(t)}
    if case["op"] == "layer_norm":
        # latents whose features have means and scales of their own
        r, w = case["rows"], case["width"]
        s = {"x": (normal(r, w) * (1.0 + 0.3 * normal(w)) + 0.5 * normal(w)).to(t), "w": (1.0 + 0.1 * normal(w)).to(t),
             "b": (0.1 * normal(w)).to(t)}
        out = w
    else:
        # weights and biases as nn.Linear's initialisation spreads them
        r, k, out = case["rows"], case["in"], case["out"]
        span = 1.0 / math.sqrt(k)
        s = {"x": normal(r, k).to(t),
             "w": ((2.0 * torch.rand(out, k, generator=gen, device="cuda") - 1.0) * span).to(t),
             "b": ((2.0 * torch.rand(out, generator=gen, device="cuda") - 1.0) * span).to(t)}
    s["res"] = normal(r, out).to(t) if case["residual"] else None
    s["dy"] = normal(r, out).to(t) if case["train"] else None
    return s


def prepare(case, seed):
    s = _given(case, seed)
    if case.get("train"):
        s.update({k: s[k].requires_grad_(True) for k in ("x", "w", "b", "res") if s[k] is not None})
    return {**s, "case": case}


def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "newton_schulz":
        m, n = min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
        # per step, half of two symmetric products and one whole one
        return {"bytes": 2 * case["count"] * m * n * size, "flops": case["count"] * 5 * (3 * m * m * n + m * m * m)}
    r, res, train = case["rows"], int(case["residual"]), int(case["train"])
    if case["op"] == "layer_norm":
        w = case["width"]
        return {"bytes": size * (r * w * (2 + res + 2 * train) + 2 * w * (1 + train)), "flops": r * w * (8 + 14 * train)}
    k, n = case["in"], case["out"]
    return {"bytes": size * (r * k * (1 + train) + r * n * (1 + res + train) + (n * k + n) * (1 + train)),
            "flops": 2 * r * n * k * (1 + 2 * train)}


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z / math.sqrt(2.0)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z / math.sqrt(2.0))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        th = torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * math.sqrt(2.0 / math.pi) * (1.0 + 0.134145 * z * z)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _plain_layer_norm(case, x, w, b, res, dy):
    t = x.dtype
    x, w, b = x.float(), w.float(), b.float()
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) * (x - mean)).mean(1, keepdim=True) + EPS)
    hat = (x - mean) * rstd
    y = hat * w + b
    y = (y if res is None else y + res.float()).to(t)
    if dy is None:
        return {"y": y}
    up = dy.float()
    g = up * w
    dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    out = {"y": y, "dx": dx.to(t), "dw": (up * hat).sum(0).to(t), "db": up.sum(0).to(t)}
    return out if res is None else {**out, "dres": dy}


def _plain_linear(case, x, w, b, res, dy):
    t = x.dtype
    x, w, b = x.float(), w.float(), b.float()
    z = x @ w.t() + b
    y = _act(z, case["act"])
    y = (y if res is None else y + res.float()).to(t)
    if dy is None:
        return {"y": y}
    dz = dy.float() * _act_slope(z, case["act"])
    out = {"y": y, "dx": (dz @ w).to(t), "dw": (dz.t() @ x).to(t), "db": dz.sum(0).to(t)}
    return out if res is None else {**out, "dres": dy}


def _quintic_step(x):
    a, b, c = QUINTIC
    gram = x @ x.transpose(1, 2).contiguous()
    return a * x + (b * gram + c * (gram @ gram)) @ x


def _plain_newton_schulz(g):
    x = g.float()
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2).contiguous() if tall else x
    x = x / (torch.sqrt((x * x).sum((1, 2), keepdim=True)) + NORM_EPS)
    x = _quintic_step(_quintic_step(_quintic_step(_quintic_step(_quintic_step(x)))))
    return {"out": (x.transpose(1, 2).contiguous() if tall else x).to(g.dtype)}


def _own_run(case, state):
    if case["op"] == "newton_schulz":
        from sgnn_amd import muon
        return {"out": muon.newton_schulz(state["g"], steps=5, coefficients=QUINTIC, eps=NORM_EPS)}
    from sgnn_amd import functional
    x, w, b, res, dy = (state[k] for k in ("x", "w", "b", "res", "dy"))
    if case["op"] == "layer_norm":
        y = functional.layer_norm(x, w, b, residual=res, eps=EPS)
    else:
        y = functional.linear(x, w, b, activation=case["act"], residual=res)
    if dy is None:
        return {"y": y}
    if res is None:
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    dx, dw, db, dres = torch.autograd.grad(y, (x, w, b, res), dy)
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db, "dres": dres}


def run(state):
    case = state["case"]
    if own:
        return _own_run(case, state)
    with torch.no_grad():
        if case["op"] == "newton_schulz":
            return _plain_newton_schulz(state["g"])
        form = _plain_layer_norm if case["op"] == "layer_norm" else _plain_linear
        return form(case, state["x"], state["w"], state["b"], state["res"], state["dy"])


def _exact_newton_schulz(g):
    """The steps as polynomials of the first Gram matrix G0: X5 = q4(G4) ... q0(G0) X0, G(k+1) = q(Gk)^2 Gk."""
    x = g.double()
    tall = x.shape[1] > x.shape[2]
    x = x.mT.contiguous() if tall else x
    x = x / (torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True) + NORM_EPS)
    gram = torch.bmm(x, x.mT.contiguous())
    eye = torch.eye(gram.shape[1], dtype=torch.float64, device=g.device).expand_as(gram)
    total = eye
    for _ in range(5):
        q = QUINTIC[0] * eye + QUINTIC[1] * gram + QUINTIC[2] * torch.bmm(gram, gram)
        total = torch.bmm(q, total)
        gram = torch.bmm(torch.bmm(q, gram), q)
    x = torch.bmm(total, x)
    return {"out": x.mT.contiguous() if tall else x}


def exact(case, seed):
    s = _given(case, seed)
    if case["op"] == "newton_schulz":
        return _exact_newton_schulz(s["g"])
    f = torch.nn.functional
    d = {k: v.double().requires_grad_(True) for k, v in s.items() if v is not None}
    if case["op"] == "layer_norm":
        y = f.layer_norm(d["x"], (case["width"],), d["w"], d["b"], EPS)
    else:
        z = f.linear(d["x"], d["w"], d["b"])
        y = {"none": lambda v: v, "relu": f.relu, "gelu": f.gelu, "gelu_tanh": lambda v: f.gelu(v, approximate="tanh"),
             "silu": f.silu}[case["act"]](z)
    y = y if s["res"] is None else y + d["res"]
    if s["dy"] is None:
        return {"y": y.detach()}
    named = {"dx": "x", "dw": "w", "db": "b", **({} if s["res"] is None else {"dres": "res"})}
    grads = torch.autograd.grad(y, [d[k] for k in named.values()], d["dy"].detach())
    return {"y": y.detach(), **dict(zip(named, grads))}
