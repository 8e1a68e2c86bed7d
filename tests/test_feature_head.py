"""The feature head on a rendered feature image, and the training iteration with it: the fused
products, the gradient norm and the clipped Adam steps run together as a user runs them."""
import copy

import pytest
import torch

from gsr_amd import trainer
from gsr_amd.feature_head import FeatureHead

gpu = pytest.mark.gpu


def _exact(head, x):
    """The head's formula in 64 bits on parameters rounded to its type; x [M, C] float64."""
    act = {"gelu": torch.nn.functional.gelu, "relu": torch.relu, "silu": torch.nn.functional.silu,
           "none": lambda t: t}[head.activation]
    params = {n: p.detach().to(head.dtype).double().requires_grad_(True)
              for n, p in head.named_parameters()}

    def lin(name, t):
        return t @ params[name + ".weight"].t() + params[name + ".bias"]

    x = act(lin("first", x))
    for i in range(len(head.blocks)):
        h = act(lin(f"blocks.{i}.gate", x)) * lin(f"blocks.{i}.up", x)
        x = lin(f"blocks.{i}.down", h) + x
    return lin("last", x), params


@gpu
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 0.06)])
@pytest.mark.parametrize("size", [(1, 1), (9, 7), (33, 40)])
def test_head_against_64_bits(dtype, tol, size):
    """Values and every gradient, as 2-norms: six roundings to the type follow each other in the
    forward and again in the backward, each at most 2^-8 relative in bfloat16: 12 x 2^-8 = 0.047,
    and 2e-5 covers 32-bit sums of at most 1320 products (1320 x 2^-24 = 8e-5 at worst, its square
    root in practice)."""
    g = torch.Generator().manual_seed(4)
    head = FeatureHead(70, width=48, blocks=2, hidden=88, dtype=dtype, generator=g)
    image = torch.randn((3,) + size, generator=g).cuda().requires_grad_(True)
    y = head(image)
    assert y.shape == size + (70,) and y.dtype == dtype
    dy = torch.randn(y.shape, generator=g).cuda().to(dtype)
    y.backward(dy)
    x = image.detach().to(dtype).double().requires_grad_(True)
    want, params = _exact(head, x.reshape(3, -1).t())
    want.backward(dy.double().reshape(want.shape))

    def near(a, b):
        return float((a.double() - b).norm()) <= tol * float(b.norm())

    assert near(y.reshape(want.shape), want)
    assert near(image.grad, x.grad)
    for n, p in head.named_parameters():
        assert near(p.grad, params[n].grad), n


@gpu
def test_some_pixels_are_rows_of_all():
    head = FeatureHead(40, width=32, blocks=1, generator=torch.Generator().manual_seed(1))
    image = torch.randn(3, 20, 30, device="cuda")
    pixels = torch.tensor([5, 599, 0, 5, 17], device="cuda")
    some = head(image, pixels)
    torch.testing.assert_close(some, head(image).reshape(600, 40)[pixels], rtol=1e-5, atol=1e-5)
    rows = head.rows(image.reshape(3, -1).t()[pixels].contiguous())
    torch.testing.assert_close(some, rows, rtol=1e-5, atol=1e-5)


def _scene(seed=3):
    from gsr_amd.model import SplatModel
    from gsr_amd.synthetic import make_cameras, make_gaussians, training_targets
    W, H = 120, 90
    m = SplatModel(make_gaussians(5000, sh_degree=3, seed=seed), device="cuda")
    cam = make_cameras(1, W, H, seed=seed)[0].to("cuda")
    gts, monos = training_targets(1, H, W, seed=2, device="cuda")
    return m, cam, gts[0], monos[0], W, H


@gpu
@pytest.mark.parametrize("sampled", [False, True])
def test_training_iteration_with_a_head(sampled):
    """The iteration takes the same step as its parts written out: render, losses, backward, one
    clipping over both parameter sets, both Adam steps."""
    import diff_gaussian_rasterization as dgr
    from gaussian_renderer import render
    from gsr_amd.losses import train_view_loss
    from gsr_amd.optim import clip_grad_norm_
    prev = dgr.deterministic()
    dgr.deterministic(True)
    try:
        states = []
        for parts in (False, True):
            m, cam, gt, mono, W, H = _scene()
            args = trainer.OptArgs(max_grad_norm=1e-3, feature_weight=0.5)
            trainer.make_trainable(m, args)
            g = torch.Generator().manual_seed(7)
            head = FeatureHead(24, width=32, blocks=1, generator=g)
            head.training_setup(1e-3)
            wide = torch.randn(H, W, 24, generator=g).cuda()
            pixels = torch.randint(0, H * W, (500,), generator=g).cuda() if sampled else None
            target = wide.reshape(-1, 24)[pixels] if sampled else wide
            bg = torch.zeros(3, device="cuda")
            if not parts:
                for it in (1, 2):
                    loss = trainer.train_iteration(m, cam, gt, mono, bg, args, it, 2.78,
                                                   feature_head=head,
                                                   gt_feature=(target, pixels) if sampled else target)
                    assert loss.shape == () and bool(torch.isfinite(loss))
                assert all(p.grad is None for p in head.parameters())
            else:
                for it in (1, 2):
                    pkg = render(cam, m, trainer._Pipe(), bg, args)
                    loss, _ = train_view_loss(pkg["render"], pkg["depth"], gt, mono,
                                              args.lambda_dssim, args.depth_weight)
                    out = head(pkg["feature"], pixels)
                    loss = loss + 0.5 * (1 - torch.nn.functional.cosine_similarity(
                        out, target, dim=-1).mean())
                    loss.backward()
                    assert float(m._language_feature.grad.abs().max()) > 0
                    clip_grad_norm_(m.parameters() + list(head.parameters()), 1e-3)
                    head.optimizer.step()
                    m.optimizer.step()
                    m.optimizer.zero_grad()
                    head.optimizer.zero_grad()
            states.append([p.detach().clone() for p in m.parameters() + list(head.parameters())])
        # the norm is taken over the same gradients in another order of tensors: its 64-bit sum may
        # round differently in the last place, nothing else may
        for a, b in zip(*states):
            torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)
    finally:
        dgr.deterministic(prev)


@gpu
def test_clipping_without_a_head_is_inside_the_step():
    """args.max_grad_norm alone: the Gaussians' step equals clipping in place and then stepping,
    and the optimizer keeps its own setting."""
    import diff_gaussian_rasterization as dgr
    prev = dgr.deterministic()
    dgr.deterministic(True)
    try:
        states = []
        for clipped in (True, False):
            m, cam, gt, mono, W, H = _scene()
            args = trainer.OptArgs(max_grad_norm=1e-3 if clipped else None)
            trainer.make_trainable(m, args)
            trainer.train_iteration(m, cam, gt, mono, torch.zeros(3, device="cuda"), args, 1, 2.78)
            assert m.optimizer.max_grad_norm is None
            assert (m.optimizer.grad_norm is not None) == clipped
            states.append([m.optimizer.state[p]["exp_avg"].clone() for p in m.parameters()])
            if clipped:
                norm = float(m.optimizer.grad_norm)
        c = 1e-3 / (norm + 1e-6)
        assert norm > 1e-3
        for a, b in zip(*states):  # the first moments are (1 - beta1) times the gradients
            torch.testing.assert_close(a, b * c, rtol=1e-5, atol=1e-12)
    finally:
        dgr.deterministic(prev)


@gpu
def test_a_failed_forward_skips_both_steps():
    """The head and the Gaussians read one snapshot of the fault word: after a failed forward
    neither moves."""
    from gsr_amd import _lib
    m, cam, gt, mono, W, H = _scene()
    args = trainer.OptArgs(max_grad_norm=1.0)
    trainer.make_trainable(m, args)
    head = FeatureHead(8, width=16, blocks=0, generator=torch.Generator().manual_seed(1))
    head.training_setup()
    for p in list(m.parameters()) + list(head.parameters()):
        p.grad = torch.full_like(p, 0.5)
    before = [p.detach().clone() for p in m.parameters() + list(head.parameters())]
    real = _lib.step_guard
    try:
        _lib.step_guard = lambda slot: slot.fill_(1.0)
        trainer._optimizer_step(m, args=args, head=head)
    finally:
        _lib.step_guard = real
    torch.cuda.synchronize()
    for a, p in zip(before, m.parameters() + list(head.parameters())):
        assert torch.equal(a, p)
    for opt in (m.optimizer, head.optimizer):
        with pytest.raises(RuntimeError, match="skipped"):
            opt.step()
        assert opt.skipped_steps == 1


@gpu
def test_batched_step_clips():
    """train_step_views with max_grad_norm: the moments are those of the unclipped step, scaled."""
    import diff_gaussian_rasterization as dgr
    from gsr_amd.pipeline import ViewPipeline
    from gsr_amd.synthetic import make_cameras
    prev = dgr.deterministic()
    dgr.deterministic(True)
    try:
        states = []
        for limit in (1e-3, None):
            m, cam, gt, mono, W, H = _scene()
            cams = [c.to("cuda") for c in make_cameras(2, W, H, seed=3)]
            args = trainer.OptArgs(max_grad_norm=limit)
            trainer.make_trainable(m, args)
            vp = ViewPipeline(torch.device("cuda"), depth=2)
            trainer.train_step_views(m, cams, [gt, gt], [mono, mono], torch.zeros(3, device="cuda"),
                                     args, 1, 2.78, vp)
            if limit:
                c = limit / (float(m.optimizer.grad_norm) + 1e-6)
                assert c < 1
            states.append([m.optimizer.state[p]["exp_avg"].clone() for p in m.parameters()])
        for a, b in zip(*states):
            torch.testing.assert_close(a, b * c, rtol=1e-5, atol=1e-12)
    finally:
        dgr.deterministic(prev)


def test_refusals():
    for bad in (dict(out_features=0), dict(width=0), dict(blocks=-1), dict(activation="tanh"),
                dict(dtype=torch.float64)):
        with pytest.raises(ValueError):
            FeatureHead(**{"out_features": 8, "device": "cpu", **bad})
    head = FeatureHead(8, width=4, blocks=1, device="cpu")
    with pytest.raises(ValueError, match="expects"):
        head(torch.zeros(4, 5, 6))
    with pytest.raises(RuntimeError, match="no CPU path"):
        head(torch.zeros(3, 5, 6))
    with pytest.raises(ValueError, match="belong together"):
        trainer.train_iteration(None, None, None, None, None, trainer.OptArgs(), 1, 1.0,
                                feature_head=head)
    assert len(copy.deepcopy(head).state_dict()) == len(head.state_dict()) == 10
