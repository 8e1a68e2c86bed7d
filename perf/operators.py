"""Cases of the feature head's products and of the clipped optimizer step.

Each case is one call that a training or serving program makes: a fused linear layer (product,
bias, activation, residual), a gated feed-forward pair (two products, activation, product of the
two), or the global gradient norm with clipping, alone or inside the Adam step.  `run` computes it
in plain torch operations in 32 bits, or (`own`) through this repository's entry points; `exact`
computes it in 64 bits from the definition.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if os.path.join(ROOT, "sdp-gs_amd") not in sys.path:
    sys.path.insert(1, os.path.join(ROOT, "sdp-gs_amd"))

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}

# rows: M, inputs: K, outputs: N (of each of the two products in a gated pair)
LISTED = [
    # a few picked points of a view decoded: nothing but latency
    dict(name="linear points fp32", op="linear", type="fp32", rows=5, inputs=512, outputs=512,
         act="relu", residual=False, bias=True, planar=False, train=False),
    # one row through a wide layer: the weights' bytes
    dict(name="linear one row fp16", op="linear", type="fp16", rows=1, inputs=4096, outputs=8192,
         act="none", residual=True, bias=True, planar=False, train=False),
    # the head's first layer on a rendered 1008x756 feature image as it lies, [3, H, W]
    dict(name="linear image fp32", op="linear", type="fp32", rows=762048, inputs=3, outputs=64,
         act="relu", residual=False, bias=True, planar=True, train=False),
    # the head's last layer in training: every pixel of that view, forward and backward
    dict(name="linear view bf16 train", op="linear", type="bf16", rows=762048, inputs=256,
         outputs=512, act="gelu", residual=False, bias=True, planar=False, train=True),
    # a residual layer with odd sizes: rows at any alignment, forward and backward
    dict(name="linear odd fp32 train", op="linear", type="fp32", rows=130001, inputs=161,
         outputs=203, act="silu", residual=True, bias=True, planar=False, train=True),
    # a large product, where the matrix cores are the bound
    dict(name="linear large bf16", op="linear", type="bf16", rows=8192, inputs=4096, outputs=4096,
         act="gelu", residual=True, bias=True, planar=False, train=False),
    # a gated pair for a handful of rows
    dict(name="gated rows fp16", op="gated", type="fp16", rows=16, inputs=2048, outputs=5504,
         act="silu", residual=False, bias=False, planar=False, train=False),
    # a gated pair at odd sizes in 32 bits
    dict(name="gated odd fp32", op="gated", type="fp32", rows=20011, inputs=193, outputs=333,
         act="gelu", residual=False, bias=True, planar=False, train=False),
    # a gated block of the head in training, a quarter of a view's pixels
    dict(name="gated view bf16 train", op="gated", type="bf16", rows=190512, inputs=256,
         outputs=512, act="silu", residual=False, bias=True, planar=False, train=True),
    # a head's gradients: many small tensors of two types, latency
    dict(name="clip head mixed", op="clip", points=0, layers=30, width=96, type="bf16",
         max_norm=1.0, norm="2"),
    # all gradients of one million Gaussians, clipped in place
    dict(name="clip 1M Gaussians", op="clip", points=1000000, layers=0, width=0, type="fp32",
         max_norm=0.5, norm="2"),
    # the Adam step of one million Gaussians and a head with the clipping in it
    dict(name="adam clipped 1M", op="adam", points=1000000, layers=6, width=256, type="fp32",
         max_norm=0.5, norm="2"),
]


def listed():
    return [dict(c) for c in LISTED]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "gated", "gated", "clip", "adam"])
    kind = rng.choice(["fp32", "fp16", "bf16"])
    if op in ("clip", "adam"):
        points = _log(rng, 1, 1000000)
        layers = rng.randint(1, 7 if op == "adam" else 24)
        width = _log(rng, 8, 256)
        return dict(op=op, points=points, layers=layers, width=width,
                    type="fp32" if op == "adam" else kind, max_norm=rng.choice([0.1, 1.0, 1e4]),
                    norm="2" if op == "adam" else rng.choice(["2", "2", "inf"]))
    wide = rng.random() < 0.4
    if wide:  # few rows, many weights
        rows, inputs, outputs = _log(rng, 1, 512), _log(rng, 256, 4096), _log(rng, 256, 6144)
    else:     # many rows, a head's widths
        rows, inputs, outputs = _log(rng, 33, 500000), _log(rng, 3, 512), _log(rng, 1, 512)
    if rng.random() < 0.5:  # sizes that layers usually have
        inputs, outputs = max(8, inputs // 8 * 8), max(8, outputs // 8 * 8)
    # no drawn case costs more than the largest listed one
    rows = max(1, min(rows, int(4e11 / (12 * inputs * outputs)),
                      int(2e9 / (4 * (2 * inputs + 3 * outputs)))))
    return dict(op=op, type=kind, rows=rows, inputs=inputs, outputs=outputs,
                act=rng.choice(["none", "relu", "gelu", "silu"] if op == "linear" else
                               ["relu", "gelu", "silu"]),
                residual=op == "linear" and rng.random() < 0.5, bias=rng.random() < 0.7,
                planar=op == "linear" and not wide and inputs <= 64, train=rng.random() < 0.5)


def _normal(gen, *shape, scale=1.0, kind=torch.float32):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(kind)


def _widths(case):
    """The shapes of a Gaussian model's leaves and of a head's layers."""
    n, w = case["points"], case["width"]
    leaves = [(n, 3), (n, 3), (n, 1, 3), (n, 15, 3), (n, 1), (n, 3), (n, 4)] if n else []
    return leaves, [s for _ in range(case["layers"]) for s in ((w, w), (w,))]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]
    if case["op"] in ("clip", "adam"):
        points, head = _widths(case)
        shapes = [(s, torch.float32) for s in points]
        # a head kept in fewer bits has its biases in 32
        shapes += [(s, kind if len(s) == 2 else torch.float32) for s in head]
        params, grads = [], []
        for i, (s, t) in enumerate(shapes):
            g = _normal(gen, *s, scale=10.0 ** (-(i % 4)) * 1e-2)
            if i < len(points):  # Gaussians that no view saw have no gradient
                g *= (torch.rand(s[:1] + (1,) * (len(s) - 1), generator=gen, device="cuda") < 0.7)
            params.append(torch.nn.Parameter(_normal(gen, *s, kind=t)))
            grads.append(g.to(t))
        for p, g in zip(params, grads):
            p.grad = g
        st = {"case": case, "params": params}
        if case["op"] == "adam":
            st["lr"], st["eps"], st["betas"], st["step"] = 1e-3, 1e-15, (0.9, 0.999), 0
            st["m"] = [torch.zeros_like(p) for p in params]
            st["v"] = [torch.zeros_like(p) for p in params]
        return st
    M, K, N = case["rows"], case["inputs"], case["outputs"]
    st = {"case": case}
    # a feature image lies channel by channel: [K, M], read as its transpose
    st["x"] = _normal(gen, K, M, kind=kind).t() if case["planar"] else _normal(gen, M, K, kind=kind)
    names = ["w", "w2"] if case["op"] == "gated" else ["w"]
    for n in names:
        st[n] = _normal(gen, N, K, scale=K ** -0.5, kind=kind)
    st["b"] = _normal(gen, N, scale=0.1, kind=kind) if case["bias"] else None
    st["b2"] = _normal(gen, N, scale=0.1, kind=kind) if case["bias"] and "w2" in st else None
    st["r"] = _normal(gen, M, N, kind=kind) if case["residual"] else None
    if case["train"]:
        st["dy"] = _normal(gen, M, N, scale=1e-2, kind=kind)
        for n in ("x", "w", "w2", "b", "b2", "r"):
            if st.get(n) is not None:
                st[n].requires_grad_(True)
    return st


# ---- the plain forms: 32 bits, rounded once at the end -------------------------------------------

def _act(z, kind):
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.7071067811865476))
    if kind == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _slope(z, kind):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "gelu":
        return (0.5 * (1.0 + torch.erf(z * 0.7071067811865476))
                + z * torch.exp(-0.5 * z * z) * 0.3989422804014327)
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _f(t):
    return None if t is None else t.detach().float()


def _plain_linear(s):
    c = s["case"]
    x, w, b, r = _f(s["x"]), _f(s["w"]), _f(s["b"]), _f(s["r"])
    z = x @ w.t()
    if b is not None:
        z = z + b
    y = _act(z, c["act"])
    if r is not None:
        y = y + r
    kind = TYPES[c["type"]]
    out = {"y": y.to(kind)}
    if c["train"]:
        dy = _f(s["dy"])
        dz = dy * _slope(z, c["act"]) if c["act"] != "none" else dy
        out["x"], out["w"] = (dz @ w).to(kind), (dz.t() @ x).to(kind)
        if b is not None:
            out["b"] = dz.sum(0).to(kind)
        if r is not None:
            out["r"] = s["dy"]
    return out


def _plain_gated(s):
    c = s["case"]
    x, w, w2, b, b2 = _f(s["x"]), _f(s["w"]), _f(s["w2"]), _f(s["b"]), _f(s["b2"])
    g, u = x @ w.t(), x @ w2.t()
    if b is not None:
        g, u = g + b, u + b2
    a = _act(g, c["act"])
    kind = TYPES[c["type"]]
    out = {"y": (a * u).to(kind)}
    if c["train"]:
        dy = _f(s["dy"])
        dg, du = dy * u * _slope(g, c["act"]), dy * a
        out["x"] = (dg @ w + du @ w2).to(kind)
        out["w"], out["w2"] = (dg.t() @ x).to(kind), (du.t() @ x).to(kind)
        if b is not None:
            out["b"], out["b2"] = dg.sum(0).to(kind), du.sum(0).to(kind)
    return out


def _plain_norm(grads, norm):
    flat = torch.cat([g.reshape(-1).float() for g in grads])
    if norm == "inf":
        return flat.abs().max()
    return flat.double().square().sum().sqrt().float()  # a long sum: 64 bits


def _plain_clip(s):
    grads = [p.grad for p in s["params"]]
    norm = _plain_norm(grads, s["case"]["norm"])
    scale = torch.clamp(s["case"]["max_norm"] / (norm + 1e-6), max=1.0)
    [g.copy_(g.float() * scale) for g in grads]
    return {"norm": norm, "grads": grads}


def _plain_adam(s):
    grads = [p.grad for p in s["params"]]
    norm = _plain_norm(grads, "2")
    scale = torch.clamp(s["case"]["max_norm"] / (norm + 1e-6), max=1.0)
    s["step"] += 1
    (b1, b2), t = s["betas"], s["step"]
    size, root = s["lr"] / (1 - b1 ** t), math.sqrt(1 - b2 ** t)

    def one(p, g, m, v):
        g = g * scale
        m.add_((g - m) * (1 - b1))
        v.mul_(b2).add_((1 - b2) * g * g)
        p.sub_(size * (m / (v.sqrt() / root + s["eps"])))

    with torch.no_grad():
        [one(*a) for a in zip(s["params"], grads, s["m"], s["v"])]
    return {"norm": norm, "p": s["params"], "m": s["m"], "v": s["v"]}


# ---- this repository's entry points ----------------------------------------------------------------

def _own(s):
    c = s["case"]
    if c["op"] == "clip":
        from gsr_amd.optim import clip_grad_norm_
        norm = clip_grad_norm_(s["params"], c["max_norm"], float(c["norm"]))
        return {"norm": norm, "grads": [p.grad for p in s["params"]]}
    if c["op"] == "adam":
        from gsr_amd.optim import FusedAdam
        if "opt" not in s:  # the optimizer lives as long as the parameters it updates
            s["opt"] = FusedAdam(s["params"], lr=s["lr"], eps=s["eps"], betas=s["betas"],
                                 max_grad_norm=c["max_norm"])
        opt = s["opt"]
        opt.step()
        st = [opt.state[p] for p in s["params"]]
        return {"norm": opt.grad_norm, "p": s["params"], "m": [e["exp_avg"] for e in st],
                "v": [e["exp_avg_sq"] for e in st]}
    from gsr_amd.linear import fused_linear, gated_linear
    if c["op"] == "linear":
        y = fused_linear(s["x"], s["w"], s["b"], activation=c["act"], residual=s["r"])
        names = ["x", "w", "b", "r"]
    else:
        y = gated_linear(s["x"], s["w"], s["w2"], s["b"], s["b2"], activation=c["act"])
        names = ["x", "w", "w2", "b", "b2"]
    out = {"y": y}
    if c["train"]:
        names = [n for n in names if s[n] is not None]
        out.update(zip(names, torch.autograd.grad(y, [s[n] for n in names], s["dy"])))
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"linear": _plain_linear, "gated": _plain_gated, "clip": _plain_clip,
                "adam": _plain_adam}[state["case"]["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    if case["op"] in ("clip", "adam"):
        points, head = _widths(case)
        size = 2 if case["type"] != "fp32" else 4
        n4 = sum(math.prod(s) for s in points) + sum(math.prod(s) for s in head if len(s) == 1)
        nt = sum(math.prod(s) for s in head if len(s) == 2)
        grad = 4 * n4 + size * nt
        if case["op"] == "clip":  # read and written once
            return {"bytes": 2 * grad, "flops": 3 * (n4 + nt)}
        return {"bytes": 7 * grad, "flops": 16 * (n4 + nt)}
    M, K, N = case["rows"], case["inputs"], case["outputs"]
    two = 2 if case["op"] == "gated" else 1
    size = 4 if case["type"] == "fp32" else 2
    weights = two * (N * K + (N if case["bias"] else 0))
    n = M * K + weights + M * N * (2 if case["residual"] else 1)
    flops = 2 * two * M * N * K
    if case["train"]:  # dy, and the gradients out
        n += M * N + M * K + weights
        flops *= 3
    return {"bytes": size * n, "flops": flops}


# ---- 64 bits, from the definitions -----------------------------------------------------------------

def _exact_act(z, kind):
    return {"relu": torch.relu, "silu": torch.nn.functional.silu,
            "gelu": torch.nn.functional.gelu, "none": lambda t: t}[kind](z)


def _exact_step(s):
    c = s["case"]
    g = [p.grad.double() for p in s["params"]]
    tops = torch.stack([torch.linalg.vector_norm(t, ord=float(c["norm"])) for t in g])
    norm = torch.linalg.vector_norm(tops, ord=float(c["norm"]))
    scale = min(1.0, c["max_norm"] / (float(norm) + 1e-6))
    g = [t * scale for t in g]
    if c["op"] == "clip":
        return {"norm": norm, "grads": g}
    (b1, b2), lr, eps = s["betas"], s["lr"], s["eps"]
    m, v = [(1 - b1) * t for t in g], [(1 - b2) * t.pow(2) for t in g]
    # the first step from zero moments: the corrected moments are g and g^2
    p = [q.detach().double() - lr * t / (t.abs() + eps) for q, t in zip(s["params"], g)]
    return {"norm": norm, "p": p, "m": m, "v": v}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("clip", "adam"):
        return _exact_step(s)
    names = [n for n in ("x", "w", "w2", "b", "b2", "r") if s.get(n) is not None]
    d = {n: s[n].detach().double().requires_grad_(bool(case["train"])) for n in names}
    with torch.set_grad_enabled(bool(case["train"])):
        a = _exact_act(torch.nn.functional.linear(d["x"], d["w"], d.get("b")), case["act"])
        if case["op"] == "gated":
            a = a * torch.nn.functional.linear(d["x"], d["w2"], d.get("b2"))
        y = a + d["r"] if "r" in d else a
    out = {"y": y.detach()}
    if case["train"]:
        y.backward(s["dy"].double())
        out.update({n: d[n].grad for n in names})
    return out
