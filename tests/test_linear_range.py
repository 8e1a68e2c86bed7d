"""Where operands or the gradients before an activation leave the range that their type, or its
parts, hold in full."""
import pytest
import torch

import linear_ref as ref
from gsr_amd.linear import fused_linear, gated_linear

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("small", ["x", "w0"])
@pytest.mark.parametrize("power", [100, 116, 124, 130])
@pytest.mark.parametrize("M,K,N", [(16, 64, 64), (3000, 64, 64), (33000, 64, 64), (33000, 3, 64),
                                   (300, 1040, 40)])
def test_small_float_operands(M, K, N, power, small):
    """A float32 operand is split into three bfloat16 parts, whose steps end at 2^-133: each operand
    is held to half of that, 2^-134, if not better, so it is the other's size that says what is lost."""
    d = ref.inputs(M + power, M, K, N, torch.float32, "cuda", bias=False)
    large = "w0" if small == "x" else "x"
    d[small], d[large] = d[small] * 2.0 ** -power, d[large].clamp(-4, 4) * 2.0 ** min(power, 118)
    got = fused_linear(d["x"], d["w0"])
    x, w = d["x"].double(), d["w0"].double()
    want = x @ w.t()
    bound = (ref.sum_error(K, x, w.t()) + ref.rounded(want, torch.float32)
             + 2.0 ** -134 * (x.abs().sum(1, keepdim=True) + w.abs().sum(1)))
    ref.check({"y": got}, {"y": (want, bound)}, f"{M}x{K}x{N} 2^-{power}")


def _grads(y, leaves, dy):
    return torch.autograd.grad(y, leaves, dy)


@gpu
@pytest.mark.parametrize("M", [40, 33000])
def test_float16_gradients_before_an_activation_have_that_types_range(M):
    """Beyond 65504 such a gradient is an infinity, and so are the products with it: the rows of dx
    that it belongs to are not finite, never a finite wrong value, the others are as they were.
    The bias gradient is summed before that rounding.  bfloat16 has float32's range."""
    K, N = 24, 16
    # every pre-activation is 2.4 (gate, up: 300), where silu's slope is 1.0998
    d = {"x": torch.ones(M, K), "w0": torch.full((N, K), 0.1), "w1": torch.full((N, K), 12.5)}
    for t in (torch.float16, torch.bfloat16):
        v = {n: a.to(t).cuda().requires_grad_(True) for n, a in d.items()}
        b = torch.zeros(N, dtype=t, device="cuda", requires_grad=True)
        for pair, top in ((False, 64000.0), (True, 500.0)):
            dy = torch.zeros(M, N, dtype=t, device="cuda")
            dy[1], dy[2], dy[3] = top, -top, 1.0  # 1 and 2 cancel in the sum over rows
            y = (gated_linear(v["x"], v["w0"], v["w1"], b, activation="silu") if pair
                 else fused_linear(v["x"], v["w0"], b, activation="silu"))
            dx, dw, db = _grads(y, (v["x"], v["w0"], b), dy)
            finite = torch.isfinite(dx).all(1)
            if t is torch.bfloat16:
                assert bool(finite.all()) and bool(torch.isfinite(dw).all())
            else:
                assert not bool(torch.isfinite(dx[1:3]).any())
                assert bool(finite[0]) and bool(finite[3:].all())
                assert not bool(torch.isfinite(dw).any())
            dy[1], dy[2] = 0, 0
            y = (gated_linear(v["x"], v["w0"], v["w1"], b, activation="silu") if pair
                 else fused_linear(v["x"], v["w0"], b, activation="silu"))
            alone = _grads(y, (v["x"], b), dy)
            assert torch.equal(dx[3:], alone[0][3:])
            # sums of +-70000 or 150000 in 32 bits beside 1 or 330: 4 of their 2^-24
            assert bool(((db - alone[1]).abs() <= 2.0 ** -5 + 2 * ref.half_step(t) * alone[1].abs()).all())


@gpu
def test_float16_gradients_below_half_a_step_are_lost_for_the_products_only():
    """2^-25 is float16's half step around 0: a gradient below it adds nothing to dx and dw; the
    bias gradient, summed from unrounded ones, has it."""
    M, K, N = 4096, 8, 16
    x = torch.zeros(M, K, dtype=torch.float16, device="cuda", requires_grad=True)
    w = torch.ones(N, K, dtype=torch.float16, device="cuda", requires_grad=True)
    b = torch.zeros(N, dtype=torch.float16, device="cuda", requires_grad=True)
    y = fused_linear(x, w, b, activation="silu")  # at 0 the slope is 1/2
    dy = torch.full((M, N), 2.0 ** -24 * 0.75, device="cuda").to(torch.float16)  # 2^-24
    dx, _, db = _grads(y, (x, w, b), dy)
    assert not bool(dx.any())
    assert bool((db == M * 2.0 ** -25).all())
