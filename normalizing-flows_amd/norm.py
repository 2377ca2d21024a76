"""Layer normalisation for conditioner networks (no reference counterpart; the reference has BatchNorm only,
made.py:232-236, resnet.py:26-31).

BatchNorm couples the samples of a batch and changes a flow's density between train() and eval(); layer normalisation
works on each sample alone.  Its statistics run over the hidden units, so it belongs into a coupling conditioner
(``ResidualNet(use_layer_norm=True)``) and not between the masked layers of a MADE, where a unit would see the units of
higher degree.
"""
import torch
from torch import nn

from . import _lib


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x (biased variance; statistics in fp32).

    x: [..., features] on the GPU, float32, bfloat16 or float16, rows at any stride; the result has its shape and type.
    weight, bias: float32 vectors of `features` elements, or None.  eps >= 0 is taken as float32.  Differentiable once, by
    backward passes (not under create_graph, nor in forward mode), in x, weight and bias; the gradients of weight and bias are
    summed in a fixed order (the same inputs give the same bits)."""
    return _lib.nodes().layer_norm(x, weight, bias, eps)


class LayerNorm(nn.Module):
    """layer_norm over the last axis with a learned weight (ones at first) and bias (zeros)."""

    def __init__(self, features, eps=1e-5, elementwise_affine=True, bias=True):
        super().__init__()
        if not isinstance(features, int) or features < 1:
            raise ValueError('features must be a positive int, got %r' % (features,))
        self.features, self.eps = features, eps
        self.weight = nn.Parameter(torch.ones(features)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(features)) if elementwise_affine and bias else None

    def forward(self, x):
        if x.dim() < 1 or x.shape[-1] != self.features:
            raise ValueError('expected a last axis of %d features, got shape %s' % (self.features, tuple(x.shape)))
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return '%d, eps=%g, elementwise_affine=%s, bias=%s' % (self.features, self.eps, self.weight is not None,
                                                               self.bias is not None)
