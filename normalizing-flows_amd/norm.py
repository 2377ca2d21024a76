"""Layer normalisation for conditioner networks (no reference counterpart; the reference has BatchNorm only,
made.py:232-236, resnet.py:26-31).

BatchNorm couples the samples of a batch and changes a flow's density between train() and eval(); layer normalisation
works on each sample alone.  Its statistics run over the hidden units, so it belongs into a coupling conditioner
(``ResidualNet(use_layer_norm=True)``) and not between the masked layers of a MADE, where a unit would see the units of
higher degree.
"""
import numbers

import torch
from torch import nn

from . import _lib


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x (biased variance; statistics in fp32).

    x: [..., features] on the GPU, float32, bfloat16 or float16, rows at any stride; the result has its shape and type.
    weight, bias: float32 vectors of `features` elements, or None.  Differentiable once in x, weight and bias; the
    gradients of weight and bias are summed in a fixed order (the same inputs give the same bits)."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError('x must be a tensor on the GPU (MI355X); this package has no CPU path')
    if x.dtype not in _lib.NF_ELEM:
        raise TypeError('x must be float32, bfloat16 or float16, got %s' % x.dtype)
    if x.dim() < 1 or not 1 <= x.shape[-1] < 2 ** 31:
        raise ValueError('x must have a last axis of at least one element, got shape %s' % (tuple(x.shape),))
    if not isinstance(eps, numbers.Real) or not 0 <= eps < float('inf'):
        raise ValueError('eps must be a finite number >= 0, got %r' % (eps,))
    rows = _lib.unit_rows(x if x.dim() == 2 else x.reshape(-1, x.shape[-1]))
    if torch.is_grad_enabled() and (x.requires_grad or any(t is not None and t.requires_grad for t in (weight, bias))):
        from .autograd import LayerNormFn
        y = LayerNormFn.apply(rows, weight, bias, float(eps))
    else:
        y = _lib.layer_norm(rows, weight, bias, float(eps))[0]
    return y.view(x.shape)


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
