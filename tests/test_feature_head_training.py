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
