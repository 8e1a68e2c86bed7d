"""Gradients of more elements than one sweep of a launch's workgroups takes (2048 x 8192)."""
import math

import pytest
import torch

from gsr_amd.optim import FusedAdam, clip_grad_norm_, grad_norm

gpu = pytest.mark.gpu
SWEEP = 2048 * 8192
KINDS = [torch.float32, torch.bfloat16, torch.float16]

# borders between tensors inside the first, second and third sweep, the last one ragged; and behind
# a launch's 128 tensors another launch with sweeps of its own
SETS = {"three sweeps": [SWEEP - 100001, 70001, SWEEP + 50003, 1, 999, SWEEP // 2 + 17],
        "two launches": [1001 + i for i in range(127)] + [SWEEP + 5, 300, SWEEP + 8193, 77]}
TOL = 2.0 ** -23  # the result's rounding to 32 bits and that of sums of 64 bits, 4 10^7 terms: 2^-27


def _grads(name):
    """Tensors of magnitudes of their own, so that one left out or taken twice shows in the sums."""
    g = torch.Generator(device="cuda").manual_seed(len(name))
    out = []
    for i, n in enumerate(SETS[name]):
        scale = 2.0 ** -(i % 5) * (SWEEP / (n + 1000)) ** 0.5
        out.append((torch.randn(n, generator=g, device="cuda") * scale * 1e-2).to(KINDS[i % 3]))
    return out


def _exact(grads, order):
    tops = torch.stack([torch.linalg.vector_norm(g.double(), ord=order) for g in grads])
    return float(torch.linalg.vector_norm(tops, ord=order))


@gpu
@pytest.mark.parametrize("order", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("name", list(SETS))
def test_norm(name, order):
    grads = _grads(name)
    for k in (None, 2, len(grads) - 2):  # the largest element in the second and in the last sweep
        if k is not None:
            grads[k][-3] = 3e4 if order == math.inf else 50.0
        want = _exact(grads, order)
        assert abs(float(grad_norm(grads, order)) - want) <= TOL * want, k


@gpu
@pytest.mark.parametrize("order", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("name", list(SETS))
def test_clip_in_place(name, order):
    grads = _grads(name)
    before = [g.clone() for g in grads]
    params = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty_like(g))
        p.grad = g
        params.append(p)
    want = _exact(grads, order)
    norm = clip_grad_norm_(params, 0.25 * want, order)
    assert abs(float(norm) - want) <= TOL * want
    c = 0.25 * want / (want + 1e-6)
    for i, (g, b) in enumerate(zip(grads, before)):
        # the factor carries the norm's rounding and two of its own; the product and the type one
        b = b.double()
        u = torch.finfo(g.dtype).eps / 2
        bound = (4 * 2.0 ** -24 + u) * c * b.abs() + (2.0 ** -25 if g.dtype == torch.float16 else 0)
        assert bool(((g.double() - c * b).abs() <= bound).all()), i


@gpu
def test_adam_with_clipping():
    """The bits of clipping in place and then stepping, over three sweeps of the norm."""
    shapes = [SWEEP + 50003, 999, SWEEP // 2 + 17, SWEEP - 100001]
    g = torch.Generator(device="cuda").manual_seed(3)
    grads = [torch.randn(n, generator=g, device="cuda") * 2.0 ** -i for i, n in enumerate(shapes)]
    pa, pb = ([torch.nn.Parameter(torch.zeros_like(t)) for t in grads] for _ in range(2))
    for p, q, t in zip(pa, pb, grads):
        p.grad, q.grad = t.clone(), t
    a, b = FusedAdam(pa, lr=1e-2), FusedAdam(pb, lr=1e-2, max_grad_norm=0.5)
    norm = clip_grad_norm_(pa, 0.5)
    a.step()
    b.step()
    assert torch.equal(norm, b.grad_norm)
    assert all(torch.equal(p, q) for p, q in zip(pa, pb))
