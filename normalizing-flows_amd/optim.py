"""Orthogonalised matrix updates for training flows (no reference counterpart; the reference trains with torch's Adam,
test2.py:127-135).

    orthogonalize : G -> X with G's singular vectors and singular values near 1, by Newton-Schulz products
    muon_update   : one Muon step over lists of weight matrices, in place
    Muon          : the torch.optim.Optimizer around it, for the weight matrices of a flow (biases and norm vectors go to
                    another optimizer)

A masked weight's gradient is zero where its mask is; the orthogonalised update of the whole matrix is not.  The masked
entries of the stored weight then move without any effect on the layer, whose kernels fold the mask in.
"""
import math
import numbers

import torch
from torch.autograd import forward_ad

from . import _lib


def _check_iteration(steps, eps):
    if not isinstance(steps, int) or isinstance(steps, bool) or not 1 <= steps <= 100:
        raise ValueError('steps must be an int from 1 to 100, got %r' % (steps,))
    _check_number('eps', eps, 0)


def _check_number(name, value, low, below=math.inf):
    if not isinstance(value, numbers.Real) or not low <= value < below:
        raise ValueError('%s must be a number in [%g, %g), got %r' % (name, low, below, value))


def _check_tangents(name, tensors):
    """A tangent of forward-mode differentiation would be dropped without a word."""
    if getattr(forward_ad, '_current_level', 0) < 0:    # (outside any: a step's 90 tensors would take 40 us)
        return
    if any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError('%s carry a tangent: there is no forward-mode derivative' % name)


def orthogonalize(matrices, steps=5, eps=1e-7):
    """X = G / (|G|_F + eps), then `steps` times X <- a X + (b S + c S S) X with S = X X^T and a, b, c = 3.4445, -4.7750,
    2.0315 (on G^T where G has more rows than columns): each singular value s goes through the odd quintic
    a s + b s^3 + c s^5, which brings all but the smallest near 1 (0.7 to 1.2) and leaves the singular vectors.

    matrices: [..., rows, cols] on the GPU, float32, bfloat16 or float16, any strides; the result has its shape and type.
    Computed to fp32 accuracy.  Not differentiable, in no mode."""
    if not isinstance(matrices, torch.Tensor) or not matrices.is_cuda:
        raise RuntimeError('matrices must be a tensor on the GPU (MI355X); this package has no CPU path')
    if matrices.dtype not in _lib.NF_ELEM:
        raise TypeError('matrices must be float32, bfloat16 or float16, got %s' % matrices.dtype)
    if matrices.dim() < 2 or not all(1 <= n <= _lib.MAX_SIDE for n in matrices.shape[-2:]):
        raise ValueError('matrices must be [..., rows, cols] with sides of 1 to %d, got shape %s'
                         % (_lib.MAX_SIDE, tuple(matrices.shape)))
    _check_iteration(steps, eps)
    _check_tangents('matrices', [matrices])
    if torch.is_grad_enabled() and matrices.requires_grad:
        raise NotImplementedError('orthogonalize has no backward kernel: call under torch.no_grad() or detach()')
    g = matrices.detach().reshape(-1, *matrices.shape[-2:])
    if not g.numel():
        return torch.empty_like(matrices, memory_format=torch.contiguous_format)
    if g.shape[2] > 1 and g.stride(2) != 1:
        g = g.contiguous()
    return _lib.orthogonalize(g, steps, float(eps)).view(matrices.shape)


def _check_matrices(name, tensors, shapes, device, contiguous):
    for t, shape in zip(tensors, shapes):
        _lib._dev(t, name)
        if t.device != device:
            raise ValueError('%s are on %s and %s: one call takes the matrices of one device' % (name, device, t.device))
        if tuple(t.shape) != shape:
            raise ValueError('%s have shape %s where the parameter has %s' % (name, tuple(t.shape), shape))
        if contiguous and not t.is_contiguous():
            raise ValueError('%s are written in place and must be contiguous' % name)


def _check_disjoint(written, read):
    """No memory that is written may overlap any other."""
    spans = sorted([(t.data_ptr(), t.data_ptr() + t.numel() * 4, True) for t in written] +
                   [(t.data_ptr(), t.data_ptr() + t.numel() * 4, False) for t in read])
    top, top_written = 0, 0                             # ends of the spans so far, and of those that are written
    for lo, hi, w in spans:
        if lo < (top if w else top_written):
            raise ValueError('params and momentum_buffers must not share memory with each other or with grads '
                             '(the same matrix twice?)')
        top = max(top, hi)
        top_written = max(top_written, hi) if w else top_written


def muon_update(params, grads, momentum_buffers, lr, momentum=0.95, nesterov=True, weight_decay=0., steps=5, eps=1e-7):
    """One Muon step of each matrix, in place:

        M <- momentum M + grad;  U = grad + momentum M (nesterov) or M;  O = orthogonalize(U, steps, eps)
        param <- (1 - lr weight_decay) param - lr sqrt(max(1, rows / cols)) O

    params, grads, momentum_buffers: sequences of float32 [rows, cols] tensors of one GPU; params and momentum_buffers
    contiguous and without common memory.  All matrices go through together, those of one shape as one batch."""
    params, grads, momenta = list(params), list(grads), list(momentum_buffers)
    if not len(params) == len(grads) == len(momenta):
        raise ValueError('%d params, %d grads and %d momentum_buffers' % (len(params), len(grads), len(momenta)))
    _check_iteration(steps, eps)
    _check_number('lr', lr, 0)
    _check_number('momentum', momentum, 0, 1)
    _check_number('weight_decay', weight_decay, 0)
    if not params:
        return
    for p in params:
        _lib._dev(p, 'params')
        if p.dim() != 2 or max(p.shape) > _lib.MAX_SIDE:
            raise ValueError('params must be matrices with sides up to %d, got shape %s' % (_lib.MAX_SIDE, tuple(p.shape)))
    shapes, device = [tuple(p.shape) for p in params], params[0].device
    _check_matrices('params', params, shapes, device, True)
    _check_matrices('grads', grads, shapes, device, False)
    _check_matrices('momentum_buffers', momenta, shapes, device, True)
    _check_tangents('params, grads or momentum_buffers', params + grads + momenta)
    some = [i for i, s in enumerate(shapes) if s[0] and s[1]]
    if len(some) < len(params):
        params, grads, momenta = ([ts[i] for i in some] for ts in (params, grads, momenta))
        if not params:
            return
    grads = [g.detach().contiguous() for g in grads]
    _check_disjoint(params + momenta, grads)
    _lib.muon_update(params, grads, momenta, float(lr), float(momentum), bool(nesterov), float(weight_decay), steps,
                     float(eps))
    # (the kernels wrote behind torch's back: saved tensors and weight packs of these parameters are stale)
    torch.autograd.graph.increment_version(params + momenta)


class Muon(torch.optim.Optimizer):
    """muon_update over the parameters' gradients; state 'momentum_buffer' (float32).  Takes weight matrices only: give
    biases and norm vectors to another optimizer.  A step captured into a graph keeps the options that it was captured with, and
    does not announce its writes: call nf.invalidate_weight_caches() after a replay before eager calls of the layers."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0., steps=5, eps=1e-7):
        _check_number('lr', lr, 0)
        _check_number('momentum', momentum, 0, 1)
        _check_number('weight_decay', weight_decay, 0)
        _check_iteration(steps, eps)
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      eps=eps))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]['params']:
            if p.dim() != 2 or p.dtype != torch.float32:
                self.param_groups.pop()
                raise ValueError('Muon takes float32 weight matrices, got %s of shape %s' % (p.dtype, tuple(p.shape)))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_device = {}
            for p in group['params']:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError('Muon does not support sparse gradients')
                state = self.state[p]
                if 'momentum_buffer' not in state:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError('the first Muon step of a parameter makes its momentum buffer, which a captured step '
                                           'would clear at every replay: take one step before capturing')
                    state['momentum_buffer'] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                by_device.setdefault(p.device, []).append((p, p.grad, state['momentum_buffer']))
            for entries in by_device.values():
                muon_update(*zip(*entries), lr=group['lr'], momentum=group['momentum'], nesterov=group['nesterov'],
                            weight_decay=group['weight_decay'], steps=group['steps'], eps=group['eps'])
        return loss
