"""Forward-mode derivatives of the fused products are refused, not dropped."""
import pytest
import torch
from torch.autograd import forward_ad

import linear_ref as ref
from gsr_amd.linear import fused_linear, gated_linear

gpu = pytest.mark.gpu


def _calls(d):
    return {"linear": (lambda v: fused_linear(v["x"], v["w0"], v["b0"], activation="silu", residual=v["r"]),
                       ("x", "w0", "b0", "r")),
            "gated": (lambda v: gated_linear(v["x"], v["w0"], v["w1"], v["b0"], v["b1"]),
                      ("x", "w0", "w1", "b0", "b1"))}


def _refused(d):
    for call, names in _calls(d).values():
        for n in names:
            with forward_ad.dual_level():
                v = {**d, n: forward_ad.make_dual(d[n], torch.ones_like(d[n]))}
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(v)


@pytest.mark.parametrize("rows", [0, 4])
def test_a_tangent_is_refused_before_any_gpu_work(rows):
    _refused(ref.inputs(1, rows, 6, 8, torch.float32, "cpu", gated_pair=True, residual=True))


@gpu
def test_a_tangent_is_refused_on_the_gpu_and_a_level_without_one_is_not():
    d = ref.inputs(2, 5, 6, 8, torch.float32, "cuda", gated_pair=True, residual=True)
    _refused(d)
    for call, _ in _calls(d).values():
        want = call(d)
        with forward_ad.dual_level():
            assert torch.equal(call(d), want)
