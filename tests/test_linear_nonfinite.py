"""Infinities, NaN and the largest floats: they come out of every kernel, forward and backward, where
64-bit arithmetic has them, and the finite results beside them are as they should be."""
import pytest
import torch

import linear_ref as ref
from gsr_amd.linear import fused_linear, gated_linear

gpu = pytest.mark.gpu
INF = float("inf")


def _marks(v):
    return torch.isnan(v), v == INF, v == -INF


@gpu
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("t", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", [(3, 70, 90), (300, 1100, 64), (33000, 20, 40), (33000, 200, 40), (20000, 264, 264)])
def test_marks(M, K, N, t, pair, act):
    d = ref.inputs(M + K, M, K, N, t, "cuda", gated_pair=pair)
    d["x"][0, 3], d["x"][1, 5], d["x"][2, 7] = INF, float("nan"), -INF
    d["w0"][4] = 0  # against an infinity: NaN
    d["w0"][6, 2] = INF
    d["b0"][8] = -INF
    if t is torch.float32:  # an operand whose first bfloat16 part is an infinity
        d["x"][M // 2, 9] = 3.4e38
        d["w0"][:, 9] *= 1e-30
    names = [n for n in ("x", "w0", "w1", "b0", "b1") if n in d]
    v = {n: a.detach().requires_grad_(True) for n, a in d.items()}
    e = {n: a.detach().double().requires_grad_(True) for n, a in d.items()}
    y = (gated_linear(v["x"], v["w0"], v["w1"], v["b0"], v["b1"], activation=act) if pair
         else fused_linear(v["x"], v["w0"], v["b0"], activation=act))
    a = ref.act(e["x"] @ e["w0"].t() + e["b0"], act)
    want = a * (e["x"] @ e["w1"].t() + e["b1"]) if pair else a
    got = dict(zip(["y"] + names, [y] + list(torch.autograd.grad(y, [v[n] for n in names], d["dy"]))))
    exact = dict(zip(["y"] + names, [want] + list(
        torch.autograd.grad(want, [e[n] for n in names], d["dy"].double()))))
    for n in got:
        for p, q in zip(_marks(got[n]), _marks(exact[n].to(t))):
            assert torch.equal(p, q), n
    # rows without such a value in their operands, columns without such a weight
    columns = [j for j in range(N) if j not in (6, 8)]
    bounds = (ref.gated(*(d[n].double()[columns] if n != "x" else d[n].double()[3:] for n in ("x", "w0", "w1", "b0", "b1")), act, t)
              if pair else ref.linear(d["x"].double()[3:], d["w0"].double()[columns], d["b0"].double()[columns], None, act, t))
    value, bound = bounds["y"]
    kept = torch.isfinite(value.to(t))  # what rounds to an infinity was compared above
    ref.check({"y": y.detach()[3:][:, columns][kept]}, {"y": (value[kept], bound[kept])})


@gpu
def test_relu_at_nan():
    """As torch.relu: NaN out, and the gradient goes through."""
    x = torch.tensor([[float("nan"), 1.0]], device="cuda")
    w = torch.eye(2, device="cuda").requires_grad_(True)
    b = torch.zeros(2, device="cuda", requires_grad=True)
    x.requires_grad_(True)
    (db,) = torch.autograd.grad(fused_linear(x, w, b, activation="relu"), b, torch.tensor([[3.0, 5.0]], device="cuda"))
    assert db.tolist() == [3.0, 5.0]
