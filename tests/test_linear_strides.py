"""Slices with gaps, odd bases and transposed memory at the sizes of every kernel: the values are
those of the formula, whatever lies in the gaps (NaN here)."""
import pytest
import torch

import linear_ref as ref
from gsr_amd.linear import fused_linear, gated_linear

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]

# rows kept in registers (1, 2, 4, 6, 8 steps of 32 inputs, ragged and whole), sums cut into ranges,
# the largest tiles, few rows, one tile
SIZES = [(32771, 20, 64), (32769, 64, 70), (33000, 100, 33), (32771, 161, 203), (32800, 256, 130),
         (300, 4100, 130), (66, 1024, 2052), (33001, 264, 264), (16500, 72, 1032), (20, 130, 1000),
         (129, 256, 257)]


def _inside(m, before, after):
    """m in the middle of a larger tensor: `before` elements of its rows and one row lie ahead."""
    big = torch.full((m.shape[0] + 2, m.shape[1] + before + after), float("nan"), dtype=m.dtype, device=m.device)
    v = big[1:-1, before:before + m.shape[1]]
    v.copy_(m)
    return v


# odd: no vector divides a base or a distance; even: gaps, but 16-byte rows wherever the sizes allow
PLACES = {"odd": lambda m: _inside(m, 3, 4), "even": lambda m: _inside(m, 8, 8 + -m.shape[1] % 8)}


@gpu
@pytest.mark.parametrize("place", list(PLACES))
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("pair", [False, True])
def test_slices(pair, M, K, N, t, place):
    d = ref.inputs(M + 3 * N, M, K, N, t, "cuda", gated_pair=pair, residual=not pair)
    want = {n: v.double() for n, v in d.items()}
    v = {n: PLACES[place](a) if a.dim() == 2 else a for n, a in d.items()}
    assert not v["x"].is_contiguous() and not v["dy"].is_contiguous()
    names = [n for n in ("x", "w0", "w1", "b0", "b1", "r") if n in d]
    for n in names:
        v[n] = v[n].detach().requires_grad_(True)
    if pair:
        y = gated_linear(v["x"], v["w0"], v["w1"], v["b0"], v["b1"], activation="silu")
        want = ref.gated(*(want[n] for n in ("x", "w0", "w1", "b0", "b1")), "silu", t, want["dy"])
    else:
        y = fused_linear(v["x"], v["w0"], v["b0"], activation="gelu", residual=v["r"])
        want = ref.linear(*(want[n] for n in ("x", "w0", "b0", "r")), "gelu", t, want["dy"])
    got = dict(zip(names, torch.autograd.grad(y, [v[n] for n in names], v["dy"])))
    got.pop("r", None)
    ref.check({"y": y.detach(), **got}, want, f"{M}x{K}x{N} {place}")


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_channel_major_slices(M, K, N, t):
    """Channel-major rows of a larger image, read in place: columns further apart than there are rows."""
    d = ref.inputs(M + 5 * N, M, K, N, t, "cuda")
    x = _inside(d["x"].t().contiguous(), 5, 2).t().detach().requires_grad_(True)
    assert x.stride() == (1, M + 7)
    w = d["w0"].detach().requires_grad_(True)
    y = fused_linear(x, w, d["b0"], activation="silu")
    dx, dw = torch.autograd.grad(y, (x, w), PLACES["odd"](d["dy"]))
    want = ref.linear(*(d[n].double() for n in ("x", "w0", "b0")), None, "silu", t, d["dy"].double())
    ref.check({"y": y.detach(), "x": dx, "w0": dw}, want, f"{M}x{K}x{N}")
