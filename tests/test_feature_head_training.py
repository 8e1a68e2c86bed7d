"""What the training of a feature head refuses, and how its step is clipped."""
import pytest
import torch

from gsr_amd import trainer
from gsr_amd.feature_head import FeatureHead

gpu = pytest.mark.gpu


def test_a_mean_over_a_view_vanishes_in_float16():
    """Why a float16 head is refused: the gradient that feature_loss gives each of its outputs, over
    as many values as a view has, is 0 in that type; bfloat16 keeps it to its rounding."""
    g = torch.Generator().manual_seed(0)
    rows, pixels, wide = 64, 762048, 512
    out, target = torch.randn(rows, wide, generator=g), torch.randn(rows, wide, generator=g)

    def gradient(t):
        y = out.to(t).detach().requires_grad_(True)
        # `rows` of the pixels that the mean is taken over
        (trainer.feature_loss(y, target) * (rows / pixels)).backward()
        return y.grad.double()

    exact = gradient(torch.float32)
    assert float(exact.norm()) > 0
    assert not gradient(torch.float16).any()
    # one rounding of the outputs and one of the gradient, each at most 2^-8 of every value
    assert float((gradient(torch.bfloat16) - exact).norm()) <= 2.0 ** -6 * float(exact.norm())


def test_a_float16_head_is_not_trained():
    head = FeatureHead(8, width=4, blocks=1, dtype=torch.float16, device="cpu")
    with pytest.raises(ValueError, match="float16"):
        head.training_setup()
    from gsr_amd.optim import FusedAdam
    head.optimizer = FusedAdam(head.parameters(), lr=1e-3)  # set up by hand: refused all the same
    with pytest.raises(ValueError, match="float16"):
        trainer.train_iteration(None, None, None, None, None, trainer.OptArgs(), 1, 1.0,
                                feature_head=head, gt_feature=torch.zeros(5, 6, 8))
    for t in (torch.float32, torch.bfloat16):
        FeatureHead(8, width=4, blocks=1, dtype=t, device="cpu").training_setup()


class _Head(torch.nn.Linear):
    def __init__(self, device, limit):
        super().__init__(3, 2, device=device)
        from gsr_amd.optim import FusedAdam
        self.optimizer = FusedAdam(self.parameters(), lr=1e-2, max_grad_norm=limit)


def _pair(device, limit, with_head):
    """A model and a head of a few parameters whose optimizers have a limit of their own."""
    from types import SimpleNamespace

    from gsr_amd.optim import FusedAdam
    g = torch.Generator().manual_seed(5)
    p = torch.nn.Parameter(torch.randn(7, 3, generator=g).to(device))
    model = SimpleNamespace(optimizer=FusedAdam([p], lr=1e-2, max_grad_norm=limit), get_xyz=p)
    head = _Head(device, limit) if with_head else None
    ps = [p] + (list(head.parameters()) if with_head else [])
    with torch.no_grad():
        for q in ps:
            q.copy_(torch.randn(q.shape, generator=g))
            q.grad = torch.randn(q.shape, generator=g).to(device)
    return model, head, ps


@pytest.mark.parametrize("with_head", [False, True])
@pytest.mark.parametrize("limit", [None, 0.5])
def test_the_arguments_limit_takes_the_place_of_the_optimizers_own(monkeypatch, with_head, limit):
    """What each optimizer's step clips by, and afterwards its own limit as before."""
    from gsr_amd import _lib, optim
    model, head, ps = _pair("cpu", 0.25, with_head)
    steps, clips = [], []
    monkeypatch.setattr(optim.FusedAdam, "step", lambda self, skip=None: steps.append((self, self.max_grad_norm)))
    monkeypatch.setattr(optim, "clip_grad_norm_", lambda params, m: clips.append((len(params), m)))
    monkeypatch.setattr(_lib, "step_guard", lambda slot: None)
    trainer._optimizer_step(model, args=trainer.OptArgs(max_grad_norm=limit), head=head)
    inside = 0.25 if limit is None else None if with_head else limit
    assert steps == ([(head.optimizer, inside)] if with_head else []) + [(model.optimizer, inside)]
    assert clips == ([(len(ps), limit)] if with_head and limit is not None else [])
    assert model.optimizer.max_grad_norm == 0.25
    assert head is None or head.optimizer.max_grad_norm == 0.25


@gpu
@pytest.mark.parametrize("with_head", [False, True])
def test_a_step_is_clipped_once(with_head):
    """With an own limit far below the arguments' the step has the bits of one without."""
    results = []
    for limit in (None, 1e-4):
        model, head, ps = _pair("cuda", limit, with_head)
        trainer._optimizer_step(model, args=trainer.OptArgs(max_grad_norm=0.5), head=head)
        opts = [model.optimizer] + ([head.optimizer] if with_head else [])
        results.append([p.detach().clone() for p in ps]
                       + [v["exp_avg"] for o in opts for v in o.state.values()])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_a_norm_is_of_the_last_step():
    """A step without clipping leaves no norm behind, one without gradients that of nothing."""
    from gsr_amd.optim import FusedAdam
    p = torch.nn.Parameter(torch.zeros(3))
    opt = FusedAdam([p], max_grad_norm=1.0)
    for limit, want in ((1.0, 0.0), (None, None)):
        opt.grad_norm = torch.tensor(7.0)
        opt.max_grad_norm = limit
        opt.step()
        assert opt.grad_norm is None if want is None else float(opt.grad_norm) == want


@gpu
def test_the_norm_of_a_step_with_a_head_is_that_of_both():
    from gsr_amd.optim import grad_norm
    model, head, ps = _pair("cuda", 1.0, True)
    want = grad_norm([q.grad for q in ps])
    trainer._optimizer_step(model, args=trainer.OptArgs(max_grad_norm=0.5), head=head)
    assert torch.equal(model.optimizer.grad_norm, want) and torch.equal(head.optimizer.grad_norm, want)
    for q in ps:
        q.grad = torch.zeros_like(q)
    trainer._optimizer_step(model, args=trainer.OptArgs(), head=head)  # each by its own limit
    assert float(model.optimizer.grad_norm) == float(head.optimizer.grad_norm) == 0.0
    model.optimizer.max_grad_norm = None
    trainer._optimizer_step(model, args=trainer.OptArgs())
    assert model.optimizer.grad_norm is None


class _PixelHead(_Head):
    """A module of one's own that is called like a FeatureHead and has its optimizer."""

    def forward(self, image, pixels=None):
        rows = image.reshape(3, -1).t()
        rows = super().forward(rows if pixels is None else rows[pixels])
        return rows if pixels is not None else rows.reshape(image.shape[1], image.shape[2], 2)


@gpu
def test_a_module_of_ones_own_as_the_head():
    from gsr_amd.model import SplatModel
    from gsr_amd.synthetic import make_cameras, make_gaussians, training_targets
    m = SplatModel(make_gaussians(500, sh_degree=3, seed=3), device="cuda")
    cam = make_cameras(1, 64, 48, seed=3)[0].to("cuda")
    gts, monos = training_targets(1, 48, 64, seed=2, device="cuda")
    args = trainer.OptArgs()
    trainer.make_trainable(m, args)
    head = _PixelHead("cuda", None)
    before = [p.detach().clone() for p in head.parameters()]
    target = torch.randn(48, 64, 2, device="cuda")
    trainer.train_iteration(m, cam, gts[0], monos[0], torch.zeros(3, device="cuda"), args, 1, 2.78,
                            feature_head=head, gt_feature=target)
    assert not any(torch.equal(a, p) for a, p in zip(before, head.parameters()))
