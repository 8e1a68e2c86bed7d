"""A bias gradient without the weights' gradient: the same bits, without the product's memory."""
import pytest
import torch

import linear_ref as ref
from gsr_amd import _lib
from gsr_amd.linear import fused_linear, gated_linear

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
NEED_DW, NEED_DB = 1, 2


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("M,K,N", [(88, 3944, 5760), (40000, 512, 512), (5, 3, 7)])
def test_scratch_is_what_is_used(kind, M, K, N):
    """Without an activation a backward has no gradient of its own to keep (dy is it), so beside the
    sums over ranges of rows (at most 512 of N each) no more than 8 columns of partial products are
    needed for the bias alone, and none of them where one range of rows is written directly."""
    L = _lib.load()
    alone = L.gsr_linear_backward_scratch_bytes(kind, M, K, N, 0, NEED_DB)
    both = L.gsr_linear_backward_scratch_bytes(kind, M, K, N, 0, NEED_DW)
    none = L.gsr_linear_backward_scratch_bytes(kind, M, K, N, 0, 0)
    ranges = min(512, -(-M // 256))
    assert none <= alone <= none + ranges * 9 * N * 4 + 256
    assert alone <= both
    if M <= 256:
        assert both <= none + 9 * N * 4 + 256
    g = L.gsr_gated_backward_scratch_bytes(kind, M, K, N, NEED_DB)
    assert g <= L.gsr_gated_backward_scratch_bytes(kind, M, K, N, NEED_DW)
    if M <= 256 and kind == 0:
        assert g <= (L.gsr_gated_backward_scratch_bytes(kind, M, K, N, 0) + 9 * 2 * N * 4 + 256)


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (200, 30, 50), (300, 7, 640), (5000, 100, 129), (16500, 72, 1032),
                                   (33001, 264, 264), (88, 700, 1500)])
def test_bias_alone(M, K, N, act, t):
    """The bias gradient alone and beside the weights' has the same bits, and is the sum it should be."""
    d = ref.inputs(M + N, M, K, N, t, "cuda")
    for image in (False, True):
        x = d["x"].t().contiguous().t() if image else d["x"]
        got = []
        for names in (("w0", "b0"), ("b0",)):
            v = {n: d[n].detach().requires_grad_(n in names) for n in ("w0", "b0")}
            y = fused_linear(x, v["w0"], v["b0"], activation=act)
            got.append(torch.autograd.grad(y, [v[n] for n in names], d["dy"]))
        assert torch.equal(got[0][-1], got[1][0]), image
    want = ref.linear(*(d[n].double() for n in ("x", "w0", "b0")), None, act, t, d["dy"].double())
    ref.check({"b0": got[1][0], "w0": got[0][0]}, want)


@gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,K,N", [(5, 3, 7), (5000, 100, 129), (33001, 264, 264), (88, 700, 1500)])
def test_both_biases_of_a_pair_alone(M, K, N, t):
    d = ref.inputs(M + N, M, K, N, t, "cuda", gated_pair=True)
    got = []
    for names in (("w0", "w1", "b0", "b1"), ("b0", "b1")):
        v = {n: d[n].detach().requires_grad_(n in names) for n in ("w0", "w1", "b0", "b1")}
        h = gated_linear(d["x"], v["w0"], v["w1"], v["b0"], v["b1"])
        got.append(torch.autograd.grad(h, [v[n] for n in names], d["dy"]))
    assert torch.equal(got[0][2], got[1][0]) and torch.equal(got[0][3], got[1][1])
    want = ref.gated(*(d[n].double() for n in ("x", "w0", "w1", "b0", "b1")), "silu", t, d["dy"].double())
    ref.check(dict(zip(("w0", "w1", "b0", "b1"), got[0])), want)
