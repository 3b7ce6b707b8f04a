"""A residual decoder of per-pixel feature rows, built from ``decoder_ops``: what turns the feature map of the index-map
rasterizer (``rasterizer2``) into colours.  The counterpart of the reference's per-pixel networks
(utils/net_utils.py, called from gaussian_renderer/__init__.py:104-210), on fused operators instead of torch's."""
import torch
import torch.nn as nn

from . import decoder_ops

NUM_FEATURES = 64  # width of a feature row of the index map


class FeatureDecoder(nn.Module):
    """``[..., in_features] -> [..., out_features]`` with values in (0, 1):

        h = gelu(lift(x))
        h = h + dropout(down(gelu(up(norm(h)))))        for every block
        y = sigmoid(head(norm(h)))

    Every line but the norms is one kernel forward.  ``dropout`` is the probability while training (``train()``); the
    masks are functions of the ``seed`` given to the call, a whole number or one int64 on the GPU (see
    ``decoder_ops.dropout``), so pass another one every step.  Everything runs in the type of the weights, which the features
    must have, also under ``torch.autocast``: for 16 bits, make or convert the decoder in that type."""

    def __init__(self, in_features=NUM_FEATURES, width=128, blocks=2, out_features=3, dropout=0.0, device=None, dtype=None):
        super().__init__()
        if not 0.0 <= dropout <= 1.0:
            raise ValueError("dropout must lie in [0, 1]")
        kw = dict(device=device, dtype=dtype)
        self.dropout = dropout
        self.lift = nn.Linear(in_features, width, **kw)
        self.norms = nn.ModuleList(nn.LayerNorm(width, **kw) for _ in range(blocks))
        self.ups = nn.ModuleList(nn.Linear(width, width, **kw) for _ in range(blocks))
        self.downs = nn.ModuleList(nn.Linear(width, width, **kw) for _ in range(blocks))
        self.head_norm = nn.LayerNorm(width, **kw)
        self.head = nn.Linear(width, out_features, **kw)

    def forward(self, features, seed=0):
        ops = decoder_ops
        h = ops.linear(features, self.lift.weight, self.lift.bias, activation="gelu")
        for i, (norm, up, down) in enumerate(zip(self.norms, self.ups, self.downs)):
            t = ops.layer_norm(h, norm.weight, norm.bias, eps=norm.eps)
            t = ops.linear(t, up.weight, up.bias, activation="gelu")
            if self.training and self.dropout > 0.0:
                t = ops.linear(t, down.weight, down.bias)
                h = ops.dropout(t, self.dropout, seed, offset=i, residual=h)
            else:
                h = ops.linear(t, down.weight, down.bias, residual=h)
        h = ops.layer_norm(h, self.head_norm.weight, self.head_norm.bias, eps=self.head_norm.eps)
        return ops.linear(h, self.head.weight, self.head.bias, activation="sigmoid")
