"""Global gradient norm and clipping (gsr_amd.optim) against 64 bits, and FusedAdam's clipping."""
import math

import pytest
import torch

from gsr_amd.optim import FusedAdam, clip_grad_norm_, grad_norm

gpu = pytest.mark.gpu
KINDS = [torch.float32, torch.float16, torch.bfloat16]


def _grads(seed, shapes, kinds=KINDS, scale=1.0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale * 10.0 ** -(i % 3)).to(kinds[i % len(kinds)]).to(device)
            for i, s in enumerate(shapes)]


def _params(grads):
    ps = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros_like(g))
        p.grad = g
        ps.append(p)
    return ps


def _exact(grads, order):
    flat = torch.cat([g.detach().double().reshape(-1).cpu() for g in grads])
    return float(torch.linalg.vector_norm(flat, ord=order))


# the result is rounded to 32 bits once (2^-24); sums in 64 bits of at most 10^6 terms add 2^-33
TOL = 2.0 ** -23

SHAPES = {"one": [(1,)], "odd": [(3,), (7, 5), (1,), (8191,), (8193,), (2, 0, 3), (33, 1, 17)],
          "splat": [(5003, 3), (5003, 1, 3), (5003, 15, 3), (5003, 1), (5003, 4)],
          "many": [(1 + 37 * i % 501,) for i in range(300)], "large": [(1 << 21,), (300001,)]}


@gpu
@pytest.mark.parametrize("order", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("shapes", list(SHAPES))
def test_norm(shapes, order):
    grads = _grads(1, SHAPES[shapes])
    n = grad_norm(grads, order)
    want = _exact(grads, order)
    assert n.dtype == torch.float32 and n.shape == () and n.is_cuda
    assert abs(float(n) - want) <= TOL * want
    assert torch.equal(n, grad_norm(grads, order))  # the same bits


@gpu
@pytest.mark.parametrize("order", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("shapes", list(SHAPES))
def test_clip_in_place(shapes, order):
    grads = _grads(2, SHAPES[shapes])
    before = [g.clone() for g in grads]
    params = _params(grads)
    want = _exact(grads, order)
    n = clip_grad_norm_(params, 0.25 * want, order)
    assert abs(float(n) - want) <= TOL * want
    c = 0.25 * want / (want + 1e-6)
    for p, g, b in zip(params, grads, before):
        assert p.grad is g
        # the factor carries the norm's rounding and two of its own; the product and the type one
        u = torch.finfo(g.dtype).eps / 2
        bound = (4 * 2.0 ** -24 + u) * c * b.double().abs() + (2.0 ** -25 if g.dtype == torch.float16 else 0)
        assert bool(((g.double() - c * b.double()).abs() <= bound).all())


@gpu
def test_small_norms_are_left_alone():
    grads = _grads(3, SHAPES["odd"])
    before = [g.clone() for g in grads]
    n = clip_grad_norm_(_params(grads), 1e6)
    assert float(n) < 1e6 and all(torch.equal(a, b) for a, b in zip(grads, before))
    clip_grad_norm_(_params(grads), math.inf)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))


@gpu
def test_max_norm_zero_and_zero_gradients():
    grads = _grads(4, [(100,), (3, 5)], [torch.float32])
    clip_grad_norm_(_params(grads), 0.0)
    assert not any(bool(g.any()) for g in grads)
    assert float(clip_grad_norm_(_params(grads), 1.0)) == 0.0
    assert not any(bool(g.any()) for g in grads)


@gpu
def test_squares_beyond_the_float_range():
    big = [torch.full((1000,), 1e30, device="cuda"), torch.full((1000,), 1e25, device="cuda")]
    assert abs(float(grad_norm(big)) / _exact(big, 2.0) - 1) <= TOL
    small = [torch.full((1000,), 1e-30, device="cuda")]
    assert abs(float(grad_norm(small)) / _exact(small, 2.0) - 1) <= TOL
    half = [torch.full((1 << 20,), 6e4, dtype=torch.float16, device="cuda")]
    assert abs(float(grad_norm(half)) / _exact(half, 2.0) - 1) <= TOL


@gpu
@pytest.mark.parametrize("order", [1.0, 2.0, math.inf])
def test_infinities_and_nan(order):
    def fresh(v):
        g = _grads(5, [(50,), (9000,)], [torch.float32])
        g[1][8500] = v
        return g
    g = fresh(float("nan"))
    assert math.isnan(float(grad_norm(g, order)))
    with pytest.raises(RuntimeError, match="non-finite"):
        clip_grad_norm_(_params(g), 1.0, order, error_if_nonfinite=True)
    assert bool(torch.isfinite(g[0]).all())  # refused: nothing was scaled
    clip_grad_norm_(_params(g), 1.0, order)
    assert all(bool(torch.isnan(t).all()) for t in g)
    g = fresh(float("-inf"))
    assert float(clip_grad_norm_(_params(g), 1.0, order)) == math.inf
    assert bool((g[0] == 0).all()) and bool(torch.isnan(g[1][8500]))


@gpu
def test_strided_gradients():
    """Transposed ones are scaled as they lie; a slice with gaps is scaled, its neighbours are not."""
    base = torch.randn(40, 60, device="cuda")
    keep = base.clone()
    p = torch.nn.Parameter(torch.zeros(60, 40, device="cuda"))
    p.grad = base.t()
    wide = torch.randn(30, 20, device="cuda")
    keep2 = wide.clone()
    q = torch.nn.Parameter(torch.zeros(30, 7, device="cuda"))
    q.grad = wide[:, 3:10]
    want = _exact([p.grad, q.grad], 2.0)
    clip_grad_norm_([p, q], 1.0)
    c = 1.0 / (want + 1e-6)
    torch.testing.assert_close(base, keep * c, rtol=6 * 2 ** -24, atol=0)
    torch.testing.assert_close(wide[:, 3:10], keep2[:, 3:10] * c, rtol=6 * 2 ** -24, atol=0)
    assert torch.equal(wide[:, :3], keep2[:, :3]) and torch.equal(wide[:, 10:], keep2[:, 10:])
    # unaligned starts: views one element into a buffer
    buf = torch.randn(20002, device="cuda", dtype=torch.bfloat16)
    keep = buf.clone()
    r = torch.nn.Parameter(torch.zeros(20000, device="cuda", dtype=torch.bfloat16))
    r.grad = buf[1:20001]
    want = _exact([r.grad], 2.0)
    assert abs(float(clip_grad_norm_(r, 1.0)) - want) <= TOL * want
    assert buf[0] == keep[0] and buf[20001] == keep[20001]


@gpu
def test_no_gradients():
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    assert float(clip_grad_norm_([p], 1.0)) == 0.0
    assert float(clip_grad_norm_([], 1.0)) == 0.0 and float(grad_norm([])) == 0.0
    p.grad = torch.zeros(3, device="cuda")
    e = torch.nn.Parameter(torch.zeros(0, 4, device="cuda"))
    e.grad = torch.zeros(0, 4, device="cuda")
    assert float(clip_grad_norm_([p, e], 1.0)) == 0.0 and float(clip_grad_norm_([e], 1.0)) == 0.0


@gpu
def test_captured_and_replayed():
    grads = _grads(6, SHAPES["splat"], [torch.float32, torch.bfloat16])
    params = _params(grads)
    clip_grad_norm_(params, 1.0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        n = clip_grad_norm_(params, 1.0)
    for k in range(4):
        new = _grads(20 + k, SHAPES["splat"], [torch.float32, torch.bfloat16])
        for a, b in zip(grads, new):
            a.copy_(b)
        g.replay()
        m = clip_grad_norm_(_params(new), 1.0)
        torch.cuda.synchronize()
        assert torch.equal(n, m) and all(torch.equal(a, b) for a, b in zip(grads, new))


@gpu
@pytest.mark.parametrize("P,limit", [(1000, 0.5), (4099, 0.5), (3000, 1e6)])
def test_adam_with_clipping_equals_clip_then_step(P, limit):
    """FusedAdam(max_grad_norm=) has the bits of clip_grad_norm_ and then a plain step, and leaves
    the gradients as they were."""
    shapes = [(P, 3), (P, 15, 3), (P, 1), (P, 4)] + [(11,)] * 20  # two launches' worth
    pa = [torch.nn.Parameter(t) for t in _grads(7, shapes, [torch.float32])]
    pb = [torch.nn.Parameter(p.detach().clone()) for p in pa]
    a = FusedAdam(pa, lr=1e-2, weight_decay=1e-2)
    b = FusedAdam(pb, lr=1e-2, weight_decay=1e-2, max_grad_norm=limit)
    assert b.grad_norm is None
    for k in range(3):
        new = _grads(30 + k, shapes, [torch.float32])
        for p, q, g in zip(pa, pb, new):
            p.grad, q.grad = g.clone(), g.clone()
        n = clip_grad_norm_(pa, limit)
        a.step()
        b.step()
        assert torch.equal(n, b.grad_norm)
        for p, q, g in zip(pa, pb, new):
            assert torch.equal(q.grad, g)
            assert torch.equal(p, q)
            assert torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"])
            assert torch.equal(a.state[p]["exp_avg_sq"], b.state[q]["exp_avg_sq"])


@gpu
def test_adam_rows_with_clipping():
    """A step in row slices takes the norm of everything when it begins."""
    shapes = [(501, 3), (501, 4)]
    pa = [torch.nn.Parameter(t) for t in _grads(8, shapes, [torch.float32])]
    pb = [torch.nn.Parameter(p.detach().clone()) for p in pa]
    for p, q, g in zip(pa, pb, _grads(9, shapes, [torch.float32])):
        p.grad, q.grad = g.clone(), g.clone()
    a, b = (FusedAdam(ps, lr=1e-2, max_grad_norm=0.1) for ps in (pa, pb))
    a.step()
    h = b.begin_rows()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.step_rows(h, 0, 200)
        b.step_rows(h, 200, None)
    torch.cuda.current_stream().wait_stream(side)
    b.end_rows(h)
    assert all(torch.equal(p, q) for p, q in zip(pa, pb))


@gpu
def test_gpu_refusals():
    g = torch.randn(10, device="cuda")
    p, q = torch.nn.Parameter(torch.zeros(10, device="cuda")), torch.nn.Parameter(torch.zeros(10, device="cuda"))
    p.grad = q.grad = g
    keep = g.clone()
    for ps in ([p, q], [p, p]):
        with pytest.raises(ValueError, match="share memory"):
            clip_grad_norm_(ps, 0.1)
    q.grad = torch.ones(1, device="cuda").expand(10)
    with pytest.raises(ValueError, match="expanded"):
        clip_grad_norm_([q], 0.1)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        grad_norm([g, g.double()])
    assert torch.equal(g, keep)


def test_refusals():
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        grad_norm([p.grad])
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_([p], bad)
        with pytest.raises(ValueError, match="max_grad_norm"):
            FusedAdam([p], max_grad_norm=bad)
    for bad in (3.0, 0.0, "fro"):
        with pytest.raises(ValueError, match="norm_type"):
            clip_grad_norm_([p], 1.0, bad)
    assert bool((p.grad == 1).all())
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        grad_norm([torch.ones(3, dtype=torch.float64)])


def test_a_refused_step_advances_nothing():
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    opt = FusedAdam([p], max_grad_norm=1.0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        opt.step()
    assert len(opt.state[p]) == 0


def test_c_entries_refuse():
    import ctypes

    from gsr_amd import _lib
    L = _lib.load()
    g, n, k = (ctypes.c_void_p * 1)(4096), (ctypes.c_int64 * 1)(4), (ctypes.c_int * 1)(0)
    bad = (ctypes.c_int * 1)(5)
    neg = (ctypes.c_int64 * 1)(-1)
    for f, args in ((L.gsr_grad_norm, (1.0, 4096, None, 4096, None)), (L.gsr_clip_grads, (1.0, 4096, 4096, None))):
        assert f(0, g, n, k, 2, *args) == f(1, g, n, k, 7, *args) == 1
        assert f(1, g, n, bad, 2, *args) == f(1, g, neg, k, 2, *args) == 1
        assert f(1, None, n, k, 2, *args) == 1
    assert L.gsr_clip_grads(1, g, n, k, 2, -1.0, 4096, 4096, None) == 1
    assert L.gsr_grad_norm(1, g, n, k, 2, 1.0, None, None, 4096, None) == 1
    assert L.gsr_grad_norm_scratch_bytes(129) == 2 * L.gsr_grad_norm_scratch_bytes(128)
