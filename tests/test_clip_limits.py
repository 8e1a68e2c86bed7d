"""Limits of the gradient norm that are no limits, wherever they come from."""
import ctypes
import math
from types import SimpleNamespace

import pytest
import torch

from gsr_amd import trainer
from gsr_amd.optim import FusedAdam

gpu = pytest.mark.gpu
BAD = [-1.0, float("nan"), -math.inf]


def _parameter(device="cpu"):
    p = torch.nn.Parameter(torch.ones(4, device=device))
    p.grad = torch.ones(4, device=device)
    return p


@pytest.mark.parametrize("bad", BAD)
def test_a_limit_set_after_construction(bad):
    p = _parameter()
    opt = FusedAdam([p])
    opt.max_grad_norm = bad
    for step in (opt.step, opt.begin_rows):
        with pytest.raises(ValueError, match="max_grad_norm"):
            step()
    assert len(opt.state[p]) == 0


@pytest.mark.parametrize("with_head", [False, True])
@pytest.mark.parametrize("bad", BAD)
def test_a_limit_from_the_training_arguments(bad, with_head):
    p = _parameter()
    model = SimpleNamespace(optimizer=FusedAdam([p]), get_xyz=p)
    head = torch.nn.Linear(2, 2)
    head.optimizer = FusedAdam(head.parameters())
    for q in head.parameters():
        q.grad = torch.ones_like(q)
    with pytest.raises(ValueError, match="max_(grad_)?norm"):
        trainer._optimizer_step(model, args=trainer.OptArgs(max_grad_norm=bad),
                                head=head if with_head else None)
    assert bool((p == 1).all()) and bool((p.grad == 1).all()) and len(model.optimizer.state[p]) == 0
    assert model.optimizer.max_grad_norm is None


@gpu
@pytest.mark.parametrize("bad", BAD)
def test_a_bad_limit_moves_nothing(bad):
    p = _parameter("cuda")
    opt = FusedAdam([p])
    opt.max_grad_norm = bad
    with pytest.raises(ValueError, match="max_grad_norm"):
        opt.step()
    assert bool((p == 1).all()) and len(opt.state[p]) == 0


@gpu
def test_the_same_gradient_with_gaps_twice_is_refused():
    """Columns of one buffer are clipped side by side, the same ones twice are not."""
    from gsr_amd.optim import clip_grad_norm_
    wide = torch.randn(30, 20, device="cuda")
    keep = wide.clone()

    def clip(*columns):
        ps = []
        for a, b in columns:
            p = torch.nn.Parameter(torch.zeros(30, b - a, device="cuda"))
            p.grad = wide[:, a:b]
            ps.append(p)
        return clip_grad_norm_(ps, 1e-3)

    for columns in (((3, 10), (3, 10)), ((3, 10), (3, 8)), ((0, 2), (3, 10), (12, 14), (3, 10))):
        with pytest.raises(ValueError, match="share memory"):
            clip(*columns)
    assert torch.equal(wide, keep)
    norm = clip((3, 10), (0, 3), (12, 20))
    c = 1e-3 / (float(norm) + 1e-6)
    torch.testing.assert_close(wide[:, :10], keep[:, :10] * c, rtol=6 * 2 ** -24, atol=0)
    torch.testing.assert_close(wide[:, 12:], keep[:, 12:] * c, rtol=6 * 2 ** -24, atol=0)
    assert torch.equal(wide[:, 10:12], keep[:, 10:12])


def test_c_entry_refuses_a_factor_from_a_bad_limit():
    """Status 1 before any GPU work where a factor is asked for; a norm alone has no limit."""
    from gsr_amd import _lib
    L = _lib.load()
    g, n, k = (ctypes.c_void_p * 1)(4096), (ctypes.c_int64 * 1)(4), (ctypes.c_int * 1)(0)
    for kind in (0, 1, 2):
        for bad in BAD:
            assert L.gsr_grad_norm(1, g, n, k, kind, bad, 4096, 4096, 4096, None) == 1
