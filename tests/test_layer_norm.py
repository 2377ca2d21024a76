"""Layer normalisation (nf.layer_norm, nf.LayerNorm, ResidualNet(use_layer_norm=True)) against the formula in 64 bits.

Tolerances are counted, not tuned.  With h = eps / 2 of the element type (one rounding of the result) and u = 2^-24 (one
fp32 rounding):
  * a row sum of the kernels has at most E adds in a thread and 22 between threads (6 in a wave, 16 waves), E <= 32 for rows up
    to 16384 elements and n / 1024 + 4 above: its error is at most (E + 22) u times the sum of magnitudes.  mu is then off by
    (E + 24) u max|x|, x - mu by that and one rounding, r (whose argument is a mean of squares) by (E + 26) u relative;
  * y = xh w + b: |dy| <= h |y| + K u [(1 + max|x| r)(1 + |xh|) |w| + |b|], K = E + 30;
  * grad_x = r (u - mean u - xh mean(u xh)): two sums more, each over products with xh:
    |dgx| <= h |gx| + 4 K u r (1 + max|x| r)(1 + max|xh|)^2 max|u|;
  * grad_w adds at most rows / 256 + 1 terms in a thread (the grid is 256 workgroups or more), 256 in a workgroup and 64 in the
    second launch: |dgw| <= (rows / 256 + 321 + K (1 + max|x| r)) u sum|g| (1 + |xh|), and grad_b likewise.
"""
import pytest
import torch
from torch import nn

import normalizing_flows_amd as nf

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def oracle(x, w, b, g, eps):
    """(y, grad_x, grad_w, grad_b, xh, r) in float64."""
    x, g = x.double(), g.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(x.shape[-1], dtype=torch.float64) if b is None else b.double()
    mu = x.mean(-1, keepdim=True)
    r = ((x - mu) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()
    xh = (x - mu) * r
    u = g * w
    gx = r * (u - u.mean(-1, keepdim=True) - xh * (u * xh).mean(-1, keepdim=True))
    return xh * w + b, gx, (g * xh).sum(0), g.sum(0), xh, r


def bounds(x, w, b, g, kind, eps=1e-5):
    y, gx, gw, gb, xh, r = oracle(x, w, b, g, eps)
    rows, n = x.shape
    h = torch.finfo(kind).eps / 2
    k = (32 if n <= 16384 else n / 1024 + 4) + 30
    wd = torch.ones(n, dtype=torch.float64) if w is None else w.double()
    bd = torch.zeros(n, dtype=torch.float64) if b is None else b.double()
    tiny = torch.finfo(kind).tiny * torch.finfo(kind).eps           # a step below the smallest normal number
    lift = 1 + x.double().abs().amax(-1, keepdim=True) * r if rows else r
    ty = h * y.abs() + k * U * (lift * (1 + xh.abs()) * wd.abs() + bd.abs()) + tiny
    top = (1 + xh.abs().amax(-1, keepdim=True)) ** 2 if rows else r
    most = (g.double() * wd).abs().amax(-1, keepdim=True) if rows else r
    tx = h * gx.abs() + 4 * k * U * r * lift * top * most + tiny
    worst = lift.max().item() if rows else 1.0
    chain = rows / 256 + 321 + k * worst
    tw = chain * U * (g.double().abs() * (1 + xh.abs())).sum(0)
    tb = chain * U * g.double().abs().sum(0)
    return (y, ty), (gx, tx), (gw, tw), (gb, tb)


def close(got, want, tol, name):
    over = (got.detach().cpu().double() - want).abs() - tol
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert bool((over <= 0).all()), (name, over.max().item())


def data(rows, n, kind, seed, offset=2.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, n, generator=gen) * 1.5 + offset * torch.randn(rows, 1, generator=gen)).to(kind)
    g = torch.randn(rows, n, generator=gen).to(kind)
    w = 1 + 0.3 * torch.randn(n, generator=gen)
    b = 0.3 * torch.randn(n, generator=gen)
    return x, w, b, g


# ---------------------------------------------------------------------------------------------- CPU: what is refused
def test_refusals():
    with pytest.raises(RuntimeError, match='GPU'):
        nf.layer_norm(torch.zeros(2, 3))
    with pytest.raises(ValueError):
        nf.LayerNorm(0)
    with pytest.raises(ValueError):
        nf.LayerNorm(4)(torch.zeros(2, 5))
    with pytest.raises(ValueError):
        nf.ResidualNet(2, 2, 8, use_batch_norm=True, use_layer_norm=True)


def test_argument_errors_before_launch():
    lib = nf._lib.load()
    one = 1 << 12                                       # (a non-NULL pointer that nothing reads: every call is refused)
    assert lib.nf_layer_norm_fwd(None, 8, None, None, None, 8, None, None, 0, 8, 1e-5, 0, None) == 0     # no rows
    assert lib.nf_layer_norm_fwd(None, 8, None, None, None, 8, None, None, 4, 8, 1e-5, 0, None) == -1
    assert lib.nf_layer_norm_fwd(one, 8, None, None, one, 8, None, None, 4, 8, 1e-5, 3, None) == -5
    assert lib.nf_layer_norm_fwd(one, 8, None, None, one, 8, None, None, 4, 0, 1e-5, 0, None) == -2
    assert lib.nf_layer_norm_fwd(one, 8, None, None, one, 8, None, None, 4, 8, -1.0, 0, None) == -2
    assert lib.nf_layer_norm_fwd(one, 8, None, None, one, 7, None, None, 4, 8, 1e-5, 0, None) == -3     # rows overlap
    assert lib.nf_layer_norm_fwd(one + 1, 8, None, None, one, 8, None, None, 4, 8, 1e-5, 1, None) == -3
    assert lib.nf_layer_norm_fwd(one, 8, None, None, one, 8, one, None, 4, 8, 1e-5, 0, None) == -1      # half the stats
    need = lib.nf_layer_norm_bwd_workspace_bytes(4, 8, 0)
    assert need >= 2 * 8 * 4
    assert lib.nf_layer_norm_bwd(one, 8, one, 8, one, one, None, one, 8, one, one, one, need - 1, 4, 8, 0, None) == -6
    assert lib.nf_layer_norm_bwd(one, 8, one, 8, None, one, None, one, 8, one, one, one, need, 4, 8, 0, None) == -1


def test_module_surface():
    net = nf.ResidualNet(3, 5, 16, num_blocks=2, use_layer_norm=True)
    keys = [k for k in net.state_dict() if 'layer_norm' in k]
    assert keys == ['blocks.%d.layer_norm_layers.%d.%s' % (b, j, p) for b in range(2) for j in range(2)
                    for p in ('weight', 'bias')]
    assert nf.LayerNorm(7, elementwise_affine=False).weight is None and nf.LayerNorm(7, bias=False).bias is None
    assert not net.hidden_stack_fusable(torch.zeros(2, 3))


# ---------------------------------------------------------------------------------------------- GPU
SHAPES = [(1, 1), (3, 1), (5, 2), (2, 7), (1, 64), (33, 63), (17, 65), (129, 256), (9, 1031), (5, 2048), (4, 2049),
          (3, 8193), (2, 16384), (3, 16385), (70, 20001), (40001, 3), (20000, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize('kind', TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize('rows,n', SHAPES)
def test_forward_and_backward(rows, n, kind):
    x, w, b, g = data(rows, n, kind, seed=rows * 7 + n)
    (y, ty), (gx, tx), (gw, tw), (gb, tb) = bounds(x, w, b, g, kind)
    xd, wd, bd = x.cuda().requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()
    out = nf.layer_norm(xd, wd, bd)
    assert out.dtype == kind
    with torch.no_grad():
        assert torch.equal(nf.layer_norm(xd, wd, bd), out)
    got = torch.autograd.grad(out, (xd, wd, bd), g.cuda())
    assert got[0].dtype == kind and got[1].dtype == torch.float32
    close(out, y, ty, 'y')
    close(got[0], gx, tx, 'grad_x')
    close(got[1], gw, tw, 'grad_w')
    close(got[2], gb, tb, 'grad_b')
    if n == 1:
        assert not got[0].any()                         # a row of one element has no gradient, exactly


@pytest.mark.gpu
@pytest.mark.parametrize('kind', TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize('n,start,pad', [(37, 1, 3), (64, 3, 1), (1031, 1, 14), (512, 0, 0)])
def test_strides_alignment_and_missing_vectors(n, start, pad, kind):
    wide, w, _, g = data(19, n + start + pad, kind, seed=n)
    x, g, w = wide[:, start:start + n], g[:, :n], w[:n]
    (y, ty), (gx, tx), (gw, tw), _ = bounds(x, w, None, g, kind)
    base = wide.cuda().requires_grad_()
    wd = w.cuda().requires_grad_()
    out = nf.layer_norm(base[:, start:start + n], wd)
    close(out, y, ty, 'y')
    got = torch.autograd.grad(out, (base, wd), g.cuda())
    close(got[0][:, start:start + n], gx, tx, 'grad_x')
    assert not got[0][:, :start].any() and not got[0][:, start + n:].any()
    close(got[1], gw, tw, 'grad_w')
    # no vectors; rows at stride 0 and a last axis that is not contiguous; a gradient expanded from one number
    xd = x[0].cuda().expand(6, n)
    close(nf.layer_norm(xd), *bounds(x[:1].expand(6, n), None, None, g[:6], kind)[0], 'expanded')
    xt = x.cuda().t().contiguous().t()
    close(nf.layer_norm(xt, wd.detach()), y, ty, 'transposed')
    leaf = x.cuda().clone().requires_grad_()
    nf.layer_norm(leaf.view(1, 19, n), wd).sum().backward()
    close(leaf.grad, *bounds(x, w, None, torch.ones(19, n, dtype=kind), kind)[1], 'sum')


@pytest.mark.gpu
def test_empty_rows_of_another_stride_keep_their_graph():
    x = torch.zeros(0, 10, device='cuda', requires_grad=True)
    nf.layer_norm(x[:, ::2]).sum().backward()
    assert x.grad.shape == (0, 10)


@pytest.mark.gpu
def test_empty_and_selected_gradients():
    w, b = torch.ones(5, device='cuda', requires_grad=True), torch.zeros(5, device='cuda', requires_grad=True)
    x = torch.zeros(0, 5, device='cuda', requires_grad=True)
    nf.layer_norm(x, w, b).sum().backward()
    assert x.grad.shape == (0, 5) and not w.grad.any() and not b.grad.any()
    x, wc, _, g = data(50, 40, torch.float32, 3)
    xd, wd = x.cuda(), wc.cuda().requires_grad_()
    (gw,) = torch.autograd.grad(nf.layer_norm(xd, wd), (wd,), g.cuda())          # no input gradient
    close(gw, *bounds(x, wc, None, g, torch.float32)[2], 'grad_w alone')
    xd.requires_grad_()
    (gx,) = torch.autograd.grad(nf.layer_norm(xd, wc.cuda()), (xd,), g.cuda())   # no sums
    close(gx, *bounds(x, wc, None, g, torch.float32)[1], 'grad_x alone')
    bd = torch.zeros(40, device='cuda', requires_grad=True)
    (gb,) = torch.autograd.grad(nf.layer_norm(xd, None, bd), (bd,), g.cuda())    # a bias without a weight
    close(gb, *bounds(x, None, bd.detach().cpu(), g, torch.float32)[3], 'grad_b alone')
    with pytest.raises(RuntimeError, match='once'):     # no second derivative
        torch.autograd.grad(nf.layer_norm(xd, wd), (xd,), g.cuda(), create_graph=True)


@pytest.mark.gpu
def test_refusals_on_the_device():
    x = torch.zeros(3, 4, device='cuda')
    for bad in (dict(weight=torch.ones(5, device='cuda')), dict(bias=torch.ones(3, device='cuda')), dict(eps=-1.0),
                dict(eps=float('nan')), dict(eps=float('inf'))):
        with pytest.raises(ValueError):
            nf.layer_norm(x, **bad)
    for bad in (dict(eps='1'), dict(weight=1.0)):
        with pytest.raises(TypeError):
            nf.layer_norm(x, **bad)
    with pytest.raises(TypeError):
        nf.layer_norm(x.double())
    with pytest.raises(TypeError):
        nf.layer_norm(x, weight=torch.ones(4, device='cuda').bfloat16())
    with pytest.raises(RuntimeError):
        nf.layer_norm(x, weight=torch.ones(4))
    with pytest.raises(ValueError):
        nf.layer_norm(torch.zeros(3, 0, device='cuda'))


@pytest.mark.gpu
def test_rows_do_not_touch_each_other_and_special_values():
    """A row of infinities or NaN stays in its row; a constant row gives the bias; the last row alone is the same bits."""
    x, w, b, _ = data(9, 130, torch.float32, 11)
    x[2, 5], x[4] = float('inf'), 3.25
    x[6, 129] = float('nan')
    out = nf.layer_norm(x.cuda(), w.cuda(), b.cuda()).cpu()
    assert out[2].isnan().all() and out[6].isnan().all()
    assert torch.equal(out[4], b)
    keep = [0, 1, 3, 4, 5, 7, 8]
    assert out[keep].isfinite().all()
    assert torch.equal(nf.layer_norm(x[8:].cuda(), w.cuda(), b.cuda()).cpu(), out[8:])


@pytest.mark.gpu
def test_large_offset_keeps_its_digits():
    """x = 1000 + noise: the second sum runs over x - mu, so the error is that of mu, not of E x^2 - mu^2."""
    x = 1000 + torch.randn(8, 512, generator=torch.Generator().manual_seed(2))
    close(nf.layer_norm(x.cuda()), *bounds(x, None, None, torch.zeros_like(x), torch.float32)[0], 'offset')


@pytest.mark.gpu
def test_streams_and_repeated_bits():
    x, w, b, g = data(3000, 200, torch.float32, 5)
    xd, wd, bd, gd = x.cuda().requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_(), g.cuda()

    def call():
        return torch.autograd.grad(nf.layer_norm(xd, wd, bd), (xd, wd, bd), gd)

    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [call() for _ in range(3)]
    again = [call() for _ in range(3)]                  # two streams at work on the same inputs
    torch.cuda.synchronize()
    for o in other + again:
        assert all(torch.equal(p, q) for p, q in zip(o, want))


@pytest.mark.gpu
def test_captured_step():
    """Forward and backward recorded into a graph, replayed on new inputs between eager calls."""
    n = 96
    x, w, b, g = (torch.zeros(257, n, device='cuda'), torch.ones(n, device='cuda'), torch.zeros(n, device='cuda'),
                  torch.zeros(257, n, device='cuda'))

    def call():
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = nf.layer_norm(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = call()
    for seed in range(4):
        for t, v in zip((x, w, b, g), data(257, n, torch.float32, seed)):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in kept]
        assert all(torch.equal(p, q) for p, q in zip(got, call()))


@pytest.mark.gpu
def test_capture_with_a_live_eager_graph_is_refused():
    """A leaf that an eager graph on another stream still holds: the forward call inside the capture says so (its backward
    pass would end the process); without that graph the same capture works."""
    m = nf.LayerNorm(40).cuda()
    x = torch.randn(30, 40, device='cuda')
    alive = m(x).sum()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match='still alive'):
            m(x)
        kept = x + 1
    graph.replay()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(x)
    graph.replay()
    torch.cuda.synchronize()
    with torch.no_grad():
        assert torch.equal(y, m(x)) and torch.equal(kept, x + 1)


def _plain_net(net, x, context=None):
    """ResidualNet(use_layer_norm=True) from its state in float64 torch operations."""
    p = {k: v.detach().cpu().double().requires_grad_() for k, v in net.named_parameters()}

    def lin(name, t):
        return t @ p[name + '.weight'].t() + p[name + '.bias']

    def norm(name, t):
        d = t - t.mean(-1, keepdim=True)
        return d / (d.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * p[name + '.weight'] + p[name + '.bias']

    h = lin('initial_layer', x if context is None else torch.cat((x, context), 1))
    for i in range(len(net.blocks)):
        at = 'blocks.%d.' % i
        t = lin(at + 'linear_layers.0', norm(at + 'layer_norm_layers.0', h).relu())
        t = lin(at + 'linear_layers.1', norm(at + 'layer_norm_layers.1', t).relu())
        h = h + (t if context is None else t * torch.sigmoid(lin(at + 'context_layer', context)))
    return lin('final_layer', h), p


@pytest.mark.gpu
@pytest.mark.parametrize('mode', ['f32', 'f16x2'])
@pytest.mark.parametrize('context', [None, 3])
def test_residual_net_with_layer_norm(context, mode):
    """Values and every parameter's gradient of the conditioner against the same network in float64.  ReLU's corners: the
    inputs are drawn so that no pre-activation lies within 1e-4 of 0, which the fp32 run cannot move across."""
    torch.manual_seed(4)
    net = nf.ResidualNet(6, 10, 32, context_features=context, num_blocks=2, use_layer_norm=True).cuda()
    with torch.no_grad():
        for p in net.parameters():
            p.add_(0.2 * torch.randn_like(p))
    x = torch.randn(64, 6)
    c = None if context is None else torch.randn(64, context)
    want, p = _plain_net(net, x.double(), None if c is None else c.double())
    g = torch.randn(64, 10)
    grads = torch.autograd.grad(want, list(p.values()), g.double())
    nf.set_matmul_dtype(mode)
    try:
        out = net(x.cuda(), None if c is None else c.cuda())
        got = torch.autograd.grad(out, list(net.parameters()), g.cuda())
        with torch.no_grad():
            again = net(x.cuda(), None if c is None else c.cuda())
    finally:
        nf.set_matmul_dtype('f32')
    # (fp32 through ten layers: 2^-24 times the about 100 roundings on a path, relative to the largest value)
    assert ((out.detach().cpu().double() - want).abs().max() / want.abs().max()).item() < 100 * U * 10
    for name, a, b in zip(p, got, grads):
        assert (a.cpu().double() - b).abs().max() <= 2e-3 * b.abs().max() + 1e-6, name
    assert torch.equal(again, out)


@pytest.mark.gpu
def test_coupling_flow_with_layer_norm_is_invertible():
    torch.manual_seed(6)
    mask = torch.arange(8) % 2
    flow = nf.BaseNeuralSplineFlow(nf.CompositeTransform([
        nf.PiecewiseRationalQuadraticCouplingTransform(
            m, lambda i, o: nf.ResidualNet(i, o, 32, use_layer_norm=True), num_bins=8, tails='linear', tail_bound=3.)
        for m in (mask, 1 - mask)]), nf.StandardNormal([8])).cuda().eval()
    x = torch.randn(300, 8).cuda()
    with torch.no_grad():
        z, lad = flow.reverse(x)
        back, lad_back = flow.forward(z)
    # (each spline's inverse is exact to fp32 roundings of values up to the tail bound)
    assert (back - x).abs().max().item() < 1e-4 and (lad + lad_back).abs().max().item() < 1e-3
    flow.train()
    loss = -flow.log_prob(x).mean()
    loss.backward()
    norms = [m for m in flow.modules() if isinstance(m, nf.LayerNorm)]
    assert len(norms) == 8 and all(m.weight.grad is not None and m.weight.grad.isfinite().all() for m in norms)


@pytest.mark.gpu
@pytest.mark.parametrize('kind', [torch.float32, torch.bfloat16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize('n', [3, 5, 37, 40, 130, 515, 1031, 2050, 8193, 16386])
def test_constant_rows_of_the_largest_values(n, kind):
    """x - mu = 0 in rows of one value (a power of two, which no sum rounds), so xh = 0, y = b, grad_w = 0, grad_b = sum g and
    grad_x = r (u - mean u) with r = 1 / sqrt(eps), however large the value is: nothing of what lies past a row's end gets in,
    where (0 - mu) r leaves fp32 (2^110 * 10^6)."""
    _, w, b, g = data(6, n, kind, n)
    x = torch.full((6, n), 2.0 ** 110).to(kind)
    x[3:] *= -1
    xd, wd, bd = x.cuda().requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()
    y = nf.layer_norm(xd, wd, bd, eps=1e-12)
    gx, gw, gb = (t.cpu() for t in torch.autograd.grad(y, (xd, wd, bd), g.cuda()))
    h = torch.finfo(kind).eps / 2
    assert torch.equal(y.detach().cpu(), b.to(kind).expand(6, n))
    assert not gw.any()
    # (sums of at most 16384 / 1024 + 22 additions a thread and between threads, those of six rows and two launches)
    k = 62
    u = g.double() * w.double()
    want, r = u - u.mean(-1, keepdim=True), 1e6
    assert bool(((gx.double() - want * r).abs() <= h * r * want.abs() + 4 * k * U * r * u.abs().amax(-1, keepdim=True)).all())
    assert bool(((gb.double() - g.double().sum(0)).abs() <= 321 * U * g.double().abs().sum(0)).all())


@pytest.mark.gpu
def test_forward_mode_is_refused():
    """A tangent is not dropped, whether or not its tensor requires a gradient; other tensors pass inside a dual level too."""
    from torch.autograd import forward_ad
    x, w, b = torch.randn(5, 8, device='cuda'), torch.ones(8, device='cuda'), torch.zeros(8, device='cuda')
    want = nf.layer_norm(x, w, b)
    with forward_ad.dual_level():
        assert torch.equal(nf.layer_norm(x, w, b), want)
        for at in range(3):
            for grad in (False, True):
                args = [t.clone().requires_grad_(grad) for t in (x, w, b)]
                args[at] = forward_ad.make_dual(args[at], torch.ones_like(args[at]))
                with pytest.raises(NotImplementedError, match='tangent'):
                    nf.layer_norm(*args)
                with torch.no_grad(), pytest.raises(NotImplementedError, match='tangent'):
                    nf.layer_norm(*args)


@pytest.mark.gpu
@pytest.mark.parametrize('held', ['outputs', 'accumulators'])
def test_capture_after_a_warm_up_whose_graph_lives(held):
    """The usual recipe: warm up on a side stream, then capture.  What the warm-up left alive - its outputs, or the gradient
    accumulators that hooks hold for good - belongs to a stream that can join the capture, so the captured step, whose gradients
    that stream accumulates, gives the eager one's values at every replay."""
    n = 72
    m, x, g = nf.LayerNorm(n).cuda(), torch.zeros(50, n, device='cuda'), torch.zeros(50, n, device='cuda')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = m(x)
        if held == 'accumulators':
            alive.backward(g)
            alive = [p.expand_as(p).grad_fn.next_functions[0][0] for p in m.parameters()]
    torch.cuda.current_stream().wait_stream(side)
    for p in m.parameters():
        p.grad = torch.ones_like(p)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for p in m.parameters():
            p.grad.zero_()
        m(x).backward(g)
    other = nf.LayerNorm(n).cuda()
    for seed in range(4):
        xs, w, b, gs = data(50, n, torch.float32, seed)
        with torch.no_grad():
            for t, v in ((x, xs), (g, gs), (m.weight, w), (m.bias, b), (other.weight, w), (other.bias, b)):
                t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = [p.grad.clone() for p in m.parameters()]
        other.zero_grad()
        other(x).backward(g)
        assert all(torch.equal(a, p.grad) for a, p in zip(got, other.parameters())), seed
    assert alive is not None


@pytest.mark.gpu
@pytest.mark.parametrize('kind', TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize('rows,n', [(70001, 64), (33000, 200), (4500, 1031), (8500, 1100), (3001, 2048), (1100, 4500), (1100, 9000),
                                    (1100, 16384), (600, 16385)])
def test_more_rows_than_workgroups(rows, n, kind):
    """Every kernel's loop over rows goes round more than once, the last time for a part of the workgroups or of their rows."""
    x, w, b, g = (t.cuda() for t in data(rows, n, kind, seed=rows + n))
    want = bounds(x, w, b, g, kind)
    xd, wd, bd = x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    out = nf.layer_norm(xd, wd, bd)
    with torch.no_grad():
        assert torch.equal(nf.layer_norm(xd, wd, bd), out)
    got = (out, *torch.autograd.grad(out, (xd, wd, bd), g))
    for name, v, (exact, tol) in zip(('y', 'grad_x', 'grad_w', 'grad_b'), got, want):
        assert bool(((v.double() - exact).abs() <= tol).all()), name
    again = torch.autograd.grad(nf.layer_norm(xd, wd, bd), (xd, wd, bd), g)
    assert all(torch.equal(p, q) for p, q in zip(got[1:], again))


@pytest.mark.gpu
@pytest.mark.parametrize('mode', ['f32', 'f16x2'])
@pytest.mark.parametrize('context', [None, 3])
def test_residual_net_away_from_the_corners_of_relu(context, mode, monkeypatch):
    """Values and every parameter's gradient of the conditioner against the same network in float64, on inputs drawn again until
    no pre-activation lies within 1e-4 of 0, across which the fp32 run cannot move: both take the same branches.

    Tolerance: ten products, norms and sums forwards and as many backwards, each of at most 64 + 22 roundings 2^-24 of a sum's
    magnitudes, which exceed the largest value by at most ten."""
    seen = []
    relu = torch.Tensor.relu
    monkeypatch.setattr(torch.Tensor, 'relu', lambda t: (seen.append(t.detach().abs().min().item()), relu(t))[1])
    torch.manual_seed(4)
    net = nf.ResidualNet(6, 10, 32, context_features=context, num_blocks=2, use_layer_norm=True).cuda()
    with torch.no_grad():
        for p in net.parameters():
            p.add_(0.2 * torch.randn_like(p))
    for _ in range(60):
        x = torch.randn(64, 6)
        c = None if context is None else torch.randn(64, context)
        seen.clear()
        want, p = _plain_net(net, x.double(), None if c is None else c.double())
        assert len(seen) == 4
        if min(seen) > 1e-4:
            break
    assert min(seen) > 1e-4
    g = torch.randn(64, 10)
    grads = torch.autograd.grad(want, list(p.values()), g.double())
    nf.set_matmul_dtype(mode)
    try:
        out = net(x.cuda(), None if c is None else c.cuda())
        got = torch.autograd.grad(out, list(net.parameters()), g.cuda())
    finally:
        nf.set_matmul_dtype('f32')
    tol = 10 * 20 * (64 + 22) * U
    assert ((out.detach().cpu().double() - want).abs().max() <= tol * want.abs().max()).item()
    for name, a, b in zip(p, got, grads):
        assert (a.cpu().double() - b).abs().max() <= tol * b.abs().max(), name
