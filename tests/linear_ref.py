"""The fused products in 64 bits, and how far a right kernel may be from them.

Bounds, per element, from the arithmetic alone (u = half a step of the result's type):
  * a sum of n products in 32 bits: (n + 10) 2^-24 sum |a||b|.  The 10 covers the bias and, where
    32-bit operands are split into three bfloat16 parts, the products of parts left out, which are
    below 4 x 2^-24 |a||b| together.
  * an activation: its slope (at most 1.13) times its argument's error, and its own evaluation:
    erf to 1.5e-7, exp and reciprocal to a few 2^-24, together below |z| 2^-21
  * its slope: the curvature (at most 0.8) times the argument's error, and 2^-20 (1 + |z|); relu's
    jumps where z is within its error of 0
  * each rounding to the type: u |value|; for float16 also half its smallest step, 2^-25.  The
    gradients before the activation are rounded for the products that follow, but not for the
    bias gradients, which are their sums.
"""
import torch

SLOPE, CURVE = 1.13, 0.8


def act(z, kind):
    return {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu,
            "gelu": torch.nn.functional.gelu}[kind](z)


def act_slope(z, kind):
    z = z.detach().clone().requires_grad_(True)
    with torch.enable_grad():
        (g,) = torch.autograd.grad(act(z, kind).sum(), z)
    return g


def half_step(t):
    return torch.finfo(t).eps / 2


def rounded(value, t):
    return half_step(t) * value.abs() + (2.0 ** -25 if t == torch.float16 else 0.0)


def sum_error(n, a, b):
    """Of a @ b with n products each."""
    return (n + 10) * 2.0 ** -24 * (a.abs() @ b.abs())


def act_error(z, ez, kind):
    return ez if kind == "none" else SLOPE * ez + z.abs() * 2.0 ** -21


def slope_error(z, ez, kind):
    if kind == "none":
        return torch.zeros_like(z)
    if kind == "relu":
        return (z.abs() <= ez).to(z.dtype)
    return CURVE * ez + 2.0 ** -20 * (1 + z.abs())


def product(x, w, b):
    """(z, its error)."""
    K = x.shape[-1]
    z = x @ w.t()
    e = sum_error(K, x, w.t())
    if b is not None:
        z, e = z + b, e + (K + 10) * 2.0 ** -24 * b.abs()
    return z, e


def gradients(dz, edz, x, ws, t, round_dz=True):
    """{name: (value, bound)} of dx, and each weight's and bias's gradient, from the pre-activation
    gradients dz[i] of products x w_i^T, within edz[i] before they are rounded."""
    M, N = dz[0].shape
    eb = edz
    if round_dz:
        edz = [e + rounded(d, t) for d, e in zip(dz, edz)]
    dx = sum(d @ w for d, w in zip(dz, ws))
    ex = sum(e @ w.abs() + sum_error(2 * N, d, w) for d, e, w in zip(dz, edz, ws))
    out = {"x": (dx, ex + rounded(dx, t))}
    for i, (d, e, f) in enumerate(zip(dz, edz, eb)):
        dw, db = d.t() @ x, d.sum(0)
        out[f"w{i}"] = (dw, e.t() @ x.abs() + sum_error(M, d.t(), x) + rounded(dw, t))
        out[f"b{i}"] = (db, f.sum(0) + (M + 10) * 2.0 ** -24 * d.abs().sum(0) + rounded(db, t))
    return out


def linear(x, w, b, r, kind, t, dy=None):
    """{name: (value, bound)}; 64-bit inputs that type t holds exactly."""
    z, ez = product(x, w, b)
    a, ea = act(z, kind), act_error(z, ez, kind)
    y = a if r is None else a + r
    out = {"y": (y, ea + 2.0 ** -23 * (a.abs() + y.abs()) + rounded(y, t))}
    if dy is not None:
        dz = dy * act_slope(z, kind)
        edz = dy.abs() * slope_error(z, ez, kind)
        if kind != "none":
            edz = edz + 2.0 ** -23 * dz.abs()
        out.update(gradients([dz], [edz], x, [w], t, kind != "none"))
    return out


def gated(x, wg, wu, bg, bu, kind, t, dh=None):
    g, eg = product(x, wg, bg)
    u, eu = product(x, wu, bu)
    a, ea = act(g, kind), act_error(g, eg, kind)
    h = a * u
    out = {"y": (h, ea * u.abs() + eu * a.abs() + ea * eu + 2.0 ** -23 * h.abs() + rounded(h, t))}
    if dh is not None:
        s, es = act_slope(g, kind), slope_error(g, eg, kind)
        dg, du = dh * u * s, dh * a
        edg = dh.abs() * (es * u.abs() + eu * s.abs() + es * eu) + 2.0 ** -22 * dg.abs()
        edu = dh.abs() * ea + 2.0 ** -23 * du.abs()
        out.update(gradients([dg, du], [edg, edu], x, [wg, wu], t))
    return out


def inputs(seed, M, K, N, t, device, gated_pair=False, bias=True, residual=False, spread=1.0):
    g = torch.Generator().manual_seed(seed)

    def make(*shape, scale=1.0):
        return (torch.randn(shape, generator=g) * scale).to(t).to(device)

    d = {"x": make(M, K, scale=spread), "w0": make(N, K, scale=K ** -0.5), "dy": make(M, N)}
    if gated_pair:
        d["w1"] = make(N, K, scale=K ** -0.5)
    if bias:
        d["b0"] = make(N)
        if gated_pair:
            d["b1"] = make(N)
    if residual:
        d["r"] = make(M, N)
    return d


def check(got, want, where=""):
    for name, value in got.items():
        w, bound = want[name]
        err = (value.double() - w).abs()
        ok = err <= bound
        assert bool(ok.all()), (
            f"{where} {name}: {int((~ok).sum())} of {ok.numel()} beyond their bound, worst ratio "
            f"{float((err / bound.clamp_min(1e-300)).max()):.3g}")
