"""A feature head on the rendered 3-channel feature (gaussian_renderer/__init__.py:280-326).

render() returns `feature` [3,H,W], the blended language feature of the Gaussians.  The features it
stands for are wider; `FeatureHead` maps each pixel (or each Gaussian's language feature) to them:

    x = act(p W_in^T + b_in)                                     in_features -> width
    x = x + (act(x W_g^T + b_g) * (x W_u^T + b_u)) W_d^T + b_d   `blocks` times, `hidden` wide
    y = x W_out^T + b_out                                        width -> out_features

built on gsr_amd.linear: one product for the first and the last layer and two for a block, the
image read as it lies ([3,H,W], no permuted copy).  Parameters are float32 (what FusedAdam
updates); `dtype` is the type the products run in.  `gsr_amd.trainer.train_iteration` trains it
with the Gaussians, in float32 or bfloat16.  A float16 head is for use only: a mean over a view's
pixels gives each output a gradient near 1 / (pixels x features), 2e-9 for 762048 x 512, below
float16's smallest step of 6e-8.  No factor on the loss helps in general: one that lifts these
gradients into the type's range can lift their sums over the pixels, the weights' gradients, out
of it.
"""
from __future__ import annotations

import torch

from .linear import ACTIVATIONS, DTYPES, fused_linear, gated_linear


class FeatureHead(torch.nn.Module):
    def __init__(self, out_features, width=256, blocks=2, hidden=None, in_features=3,
                 activation="gelu", dtype=torch.float32, device="cuda", generator=None):
        super().__init__()
        hidden = 2 * width if hidden is None else hidden
        if min(out_features, width, hidden, in_features) < 1 or blocks < 0:
            raise ValueError("FeatureHead: sizes must be at least 1 (blocks at least 0)")
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, not {activation!r}")
        if dtype not in DTYPES:
            raise ValueError(f"float32, float16 or bfloat16 expected, not {dtype}")
        self.in_features, self.out_features = in_features, out_features
        self.activation, self.dtype = activation, dtype

        def layer(n, k):
            w = torch.randn((n, k), generator=generator) * k ** -0.5
            return torch.nn.ParameterDict({"weight": torch.nn.Parameter(w.to(device)),
                                           "bias": torch.nn.Parameter(torch.zeros(n, device=device))})

        self.first = layer(width, in_features)
        self.blocks = torch.nn.ModuleList(
            torch.nn.ModuleDict({"gate": layer(hidden, width), "up": layer(hidden, width),
                                 "down": layer(width, hidden)}) for _ in range(blocks))
        self.last = layer(out_features, width)

    def _pair(self, layer):
        return layer["weight"].to(self.dtype), layer["bias"].to(self.dtype)

    def rows(self, x):
        """[..., in_features] -> [..., out_features] in `dtype`."""
        x = fused_linear(x.to(self.dtype), *self._pair(self.first), activation=self.activation)
        for b in self.blocks:
            (wg, bg), (wu, bu) = self._pair(b["gate"]), self._pair(b["up"])
            h = gated_linear(x, wg, wu, bg, bu, activation=self.activation)
            x = fused_linear(h, *self._pair(b["down"]), residual=x)
        return fused_linear(x, *self._pair(self.last))

    def forward(self, image, pixels=None):
        """A rendered feature image [in_features,H,W] -> [H,W,out_features]; with `pixels` (int64
        [S], indices into H*W) only those, [S,out_features]."""
        if image.dim() != 3 or image.shape[0] != self.in_features:
            raise ValueError(f"FeatureHead expects [{self.in_features},H,W], not {tuple(image.shape)}")
        flat = image.reshape(self.in_features, -1)
        if pixels is not None:
            return self.rows(flat[:, pixels].t())
        return self.rows(flat.t()).reshape(image.shape[1], image.shape[2], self.out_features)

    def refuse_training(self):
        """Raise ValueError if this head's type cannot hold a view's gradients."""
        if self.dtype is torch.float16:
            raise ValueError("FeatureHead: a float16 head is not trained here, the gradients of a "
                             "mean over pixels vanish in that type; use bfloat16 or float32")

    def training_setup(self, lr=1e-3):
        """The head's own FusedAdam (its parameters are not Gaussians: densification must not see
        them in the model's groups)."""
        from .optim import FusedAdam
        self.refuse_training()
        self.optimizer = FusedAdam(self.parameters(), lr=lr, eps=1e-15)
        return self.optimizer
