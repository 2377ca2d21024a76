"""nf.orthogonalize, nf.muon_update and nf.Muon against the formula in 64 bits.

Tolerance: the iteration lifts an error of a step by up to 3.98 per step (the largest slope of its polynomial), so it is
counted by running it.  `spread` runs the iteration in float64 a second time with every stored value and every product
moved by the roundings that the kernels make there, drawn at random:
  * X, S and b S + c S S are kept as two fp16 terms, a step of 2^-22 of the value (root mean square of its rounding: a step
    over sqrt 12), and the products leave out lo lo, 2^-22 / 12 of a product: 0.3 * 2^-22 together;
  * a product over K is 3 K / 16 fp32 accumulations of 16 terms each, one rounding (2^-23 / sqrt 12 = 0.58 * 2^-24) of the
    running sum each; sums of one sign grow with the result, others like the root of the sum of squares:
    0.58 * 2^-24 sqrt(3 K / 16 + 16) (|C| + sqrt((P P) (Q Q)^T)).
Independent roundings of this size give a Frobenius distance like `spread`'s; four times it is the tolerance, plus half a
step of the result's type.  Where three and two steps go through the smaller side at once (16-bit results and the Muon step)
the largest singular values cancel to a^-3 of the parts that make them up: 40.9 times a step's rounding 2^-24 on them is added."""
import ctypes
import math

import pytest
import torch

import normalizing_flows_amd as nf

A, B, C = 3.4445, -4.7750, 2.0315
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def iterate(g, steps=5, eps=1e-7, gen=None):
    """The formula in float64 on the device; with `gen`, moved by the rounding model of the kernels."""
    g = g.double()
    if g.shape[-2] > g.shape[-1]:
        return iterate(g.mT, steps, eps, gen).mT

    def noise(like):
        return torch.randn(like.shape, dtype=torch.float64, device=like.device, generator=gen)

    def kept(x):
        return x if gen is None else x * (1 + 0.3 * 2.0 ** -22 * noise(x))

    def times(p, q):
        c = p @ q
        if gen is None:
            return c
        k = p.shape[-1]
        return c + 0.58 * 2.0 ** -24 * math.sqrt(3 * k / 16 + 16) * (c.abs() + ((p * p) @ (q * q)).sqrt()) * noise(c)

    x = kept(g / (g.norm(dim=(-2, -1), keepdim=True) + eps))
    for _ in range(steps):
        s = kept(times(x, x.mT.contiguous()))
        r = kept(B * s + C * times(s, s))
        x = kept(A * x + times(r, x))
    return x


def norm(x):
    return x.double().flatten(-2).norm(dim=-1)


def tolerance(g, want, kind, steps=5, eps=1e-7, blocks=False):
    gen = torch.Generator(device=g.device).manual_seed(77)
    spread = norm(iterate(g, steps, eps, gen) - want)
    n = want.shape[-2] * want.shape[-1]
    tiny = torch.finfo(kind).tiny * torch.finfo(kind).eps * math.sqrt(n)
    if blocks or kind != torch.float32:
        spread = spread + 40.9 * 2.0 ** -24 * norm(want)
    return 4 * spread + torch.finfo(kind).eps / 2 * norm(want) + tiny


def check(got, g, kind, steps=5, eps=1e-7):
    want = iterate(g, steps, eps)
    assert got.shape == g.shape and got.dtype == kind
    over = norm(got.double() - want) - tolerance(g, want, kind, steps, eps)
    assert bool((over <= 0).all()), over.max().item()


def gradients(shape, seed, scale=1e-3, device='cuda'):
    """A few strong directions over a noise floor."""
    *batch, m, n = shape
    gen = torch.Generator().manual_seed(seed)
    rank = max(1, min(m, n) // 8)
    g = torch.randn(*batch, m, rank, generator=gen) @ torch.randn(*batch, rank, n, generator=gen) / math.sqrt(rank)
    return (scale * (g + 0.1 * torch.randn(*batch, m, n, generator=gen))).to(device)


# ---------------------------------------------------------------------------------------------- CPU: what is refused
def test_refusals():
    with pytest.raises(RuntimeError, match='GPU'):
        nf.orthogonalize(torch.zeros(2, 3))
    p = torch.nn.Parameter(torch.zeros(3))
    with pytest.raises(ValueError):
        nf.Muon([p])
    with pytest.raises(ValueError):
        nf.Muon([torch.nn.Parameter(torch.zeros(2, 3, dtype=torch.float64))])
    m = torch.nn.Parameter(torch.zeros(2, 3))
    for bad in (dict(lr=-1.), dict(momentum=1.), dict(momentum=-0.1), dict(weight_decay=float('nan')), dict(steps=0),
                dict(steps=2.5), dict(eps=float('inf'))):
        with pytest.raises(ValueError):
            nf.Muon([m], **bad)
    with pytest.raises(ValueError):
        nf.muon_update([m], [m], [], 0.1)
    with pytest.raises(RuntimeError, match='GPU'):
        nf.muon_update([m], [m], [m], 0.1)
    nf.muon_update([], [], [], 0.1)                     # nothing to do
    opt = nf.Muon([m])
    with pytest.raises(ValueError):
        opt.add_param_group({'params': [p]})
    assert len(opt.param_groups) == 1
    opt.step()                                          # no gradients: nothing happens


def test_argument_errors_before_launch():
    lib = nf._lib.load()
    one = 1 << 12                                       # (a non-NULL pointer that nothing reads: every call is refused)
    need = lib.nf_orthogonalize_workspace_bytes(2, 33, 700, 0)
    # norms; X and twice X^T of 2 x 22 cells, S and B of 2 x 2 cells, 4 KB each
    assert need == 2 * 256 * 8 + 2 * (3 * 44 + 2 * 4) * 4096
    assert lib.nf_orthogonalize_workspace_bytes(0, 3, 3, 0) == 0
    assert lib.nf_orthogonalize_workspace_bytes(1, 0, 3, 0) == 0 and lib.nf_orthogonalize_workspace_bytes(1, 3, 2 ** 20 + 1, 0) == 0
    assert lib.nf_orthogonalize_workspace_bytes(1, 3, 3, 3) == 0

    def call(g=one, ms=33 * 700, rs=700, out=one, oms=33 * 700, ors=700, ws=one, nbytes=need, count=2, rows=33, cols=700, steps=5,
             eps=1e-7, elem=0):
        return lib.nf_orthogonalize(g, ms, rs, out, oms, ors, ws, nbytes, count, rows, cols, steps, eps, elem, None)

    assert call(count=0) == 0
    assert call(elem=3) == -5
    assert call(rows=0) == -2 and call(steps=0) == -2 and call(eps=-1.0) == -2 and call(count=65536) == -2
    assert call(g=None) == -1 and call(out=None) == -1 and call(ws=None) == -1
    assert call(ors=699) == -3 and call(oms=33 * 700 - 1) == -3 and call(g=one + 2) == -3 and call(ws=one + 8) == -3
    assert call(nbytes=need - 1) == -6


def test_muon_workspace_is_bounded():
    lib = nf._lib.load()

    def need(count, side):
        sides = (ctypes.c_int * count)(*[side] * count)
        return lib.nf_muon_workspace_bytes(sides, sides, count)

    # 16 matrices of 2^14 cells, eight matrices of that size each: 8 GiB; more matrices go in sequences of 16
    assert 0 < need(1, 4096) < need(8, 4096) < need(16, 4096) == need(17, 4096) == need(200, 4096) < 9 << 30
    assert need(1, 32768) > 8 << 30


def test_overlap_check():
    from normalizing_flows_amd.optim import _check_disjoint
    t = torch.zeros(40)
    _check_disjoint([t[:10], t[10:20]], [t[20:30], t[25:40], t[20:30]])         # what is only read may overlap
    for written, read in (([t[:10], t[9:12]], []), ([t[:10], t[:10]], []), ([t[5:10]], [t[:6]]), ([t[:6]], [t[5:10]]),
                          ([t[30:35]], [t[:40], t[1:2]]), ([t[0:20], t[2:3]], [])):
        with pytest.raises(ValueError):
            _check_disjoint(written, read)


# ---------------------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize('kind', TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize('shape', [(1, 1), (1, 7), (7, 1), (2, 3), (31, 33), (32, 32), (2, 33, 129), (129, 33), (64, 64),
                                   (3, 65, 640), (1000, 300), (2, 517, 1031), (5, 40, 50, 30), (700, 17, 5), (40, 8000), (3, 32, 700), (900, 31), (5, 40000), (2, 2000, 12), (3, 96, 100), (128, 128), (288, 64), (96, 190), (33, 97), (60, 200), (120, 129), (2, 50, 3000), (1500, 100), (128, 700),
                                   (20, 512, 512)], ids=str)
def test_orthogonalize(shape, kind):
    g = gradients(shape, sum(shape)).to(kind)
    out = nf.orthogonalize(g)
    check(out, g, kind)
    assert torch.equal(nf.orthogonalize(g), out)        # the same bits again


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(130, 3000), (7000, 700), (2000, 4000), (2, 1500, 1490), (24, 390, 300), (64, 512, 500)], ids=str)
def test_tiles_and_parts(shape):
    """Sides at which the products take small and large tiles, whole k loops and parts of them."""
    g = gradients(shape, 3)
    check(nf.orthogonalize(g), g, torch.float32)


@pytest.mark.gpu
def test_large_matrix():
    g = gradients((2500, 3001), 5)
    check(nf.orthogonalize(g), g, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(70, 90), (20, 300), (150, 140), (80, 700)], ids=str)
def test_steps_eps_and_scale(shape):
    g = gradients(shape, 1)
    for steps in (1, 2, 7):
        check(nf.orthogonalize(g, steps=steps), g, torch.float32, steps=steps)
    check(nf.orthogonalize(g, eps=0.5), g, torch.float32, eps=0.5)
    for scale in (1e-34, 1e-20, 1e18, 1e34):            # squares leave the range of fp32
        h = g * 1e3 * scale
        check(nf.orthogonalize(h, eps=0.0), h, torch.float32, eps=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(200, 2000), (256, 1024), (1000, 384)], ids=str)
def test_wide_fp32_keeps_the_digits_of_single_steps(shape):
    """float32 results of wide matrices whose singular values fall over two decades: of the five steps only the first two, where
    those are still small, may go through the smaller side at once.  Late values lie near 1 and cancel to a^-2 of the parts that
    make them up, so a late block would lift a rounding of these parts by up to a^2 = 11.9.  The measure is the formula in torch's
    fp32 products: they round K sums a product where the kernels round 3 K / 16, and both keep 23 to 24 bits of each matrix, so
    step by step the kernels lose less; half as much again is allowed for the first block."""
    gen = torch.Generator().manual_seed(5)
    m, n = min(shape), max(shape)
    u, v = (torch.linalg.qr(torch.randn(k, m, generator=gen, dtype=torch.float64))[0] for k in (m, n))
    g = ((u * 10 ** (-2 * torch.arange(m) / m)) @ v.T).float().cuda()
    g = g if shape[0] == m else g.T.contiguous()
    want = iterate(g)
    x = g if shape[0] == m else g.T.contiguous()
    x = x / (x.norm() + 1e-7)
    for _ in range(5):
        s = x @ x.T
        x = A * x + (B * s + C * s @ s) @ x
    plain = norm((x if shape[0] == m else x.T) - want)
    assert norm(nf.orthogonalize(g) - want) <= 1.5 * plain


@pytest.mark.gpu
def test_singular_values_come_near_one():
    g = torch.randn(96, 200, generator=torch.Generator().manual_seed(3)).cuda()
    s = torch.linalg.svdvals(nf.orthogonalize(g).double().cpu())
    # (the quintic's fifth iterate of singular values in [0.05, 1] lies in [0.68, 1.2])
    assert 0.65 < s.min().item() and s.max().item() < 1.21


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(5, 20, 70), (5, 700, 9), (5, 40, 70), (5, 130, 150), (5, 70, 900)], ids=str)
def test_special_values_stay_in_their_matrix(shape):
    g = gradients(shape, 2)
    want = nf.orthogonalize(g)
    h = g.clone()
    h[1] = 0
    h[2, -1, -1] = float('nan')
    h[3, 0, 0] = float('inf')
    out = nf.orthogonalize(h)
    assert torch.equal(out[0], want[0]) and torch.equal(out[4], want[4])
    assert not out[1].any()
    assert out[2].isnan().all() and out[3].isnan().all()
    assert nf.orthogonalize(torch.zeros(0, 3, 4, device='cuda')).shape == (0, 3, 4)


@pytest.mark.gpu
@pytest.mark.parametrize('kind', TYPES, ids=lambda t: str(t)[6:])
def test_strides(kind):
    g = gradients((3, 50, 77), 4).to(kind)
    want = nf.orthogonalize(g)
    wide = torch.zeros(3, 52, 90, dtype=kind, device='cuda')
    wide[:, 1:51, 5:82] = g
    assert torch.equal(nf.orthogonalize(wide[:, 1:51, 5:82]), want)
    assert torch.equal(nf.orthogonalize(g.mT.contiguous().mT), want)
    assert torch.equal(nf.orthogonalize(g[1].expand(4, 50, 77)), want[1].expand(4, 50, 77))
    assert torch.equal(nf.orthogonalize(g.flip(0)[1]), want[1])
    # the transposed matrix has the transposed result (both go through the same products)
    assert torch.equal(nf.orthogonalize(g.mT), want.mT)


@pytest.mark.gpu
def test_a_batch_is_cut_where_its_workspace_ends(monkeypatch):
    g = gradients((7, 40, 33), 6)
    want = nf.orthogonalize(g)
    monkeypatch.setattr(nf._lib, 'WORKSPACE_BYTES', 3 * nf._lib.load().nf_orthogonalize_workspace_bytes(1, 40, 33, 0))
    assert torch.equal(nf.orthogonalize(g), want)
    monkeypatch.setattr(nf._lib, 'WORKSPACE_BYTES', 1)
    assert torch.equal(nf.orthogonalize(g), want)


@pytest.mark.gpu
def test_refusals_on_the_device():
    g = torch.zeros(3, 4, device='cuda')
    for bad in (dict(steps=0), dict(steps=101), dict(steps=True), dict(eps=-1.), dict(eps=float('nan'))):
        with pytest.raises(ValueError):
            nf.orthogonalize(g, **bad)
    with pytest.raises(ValueError):
        nf.orthogonalize(g[0])
    with pytest.raises(ValueError):
        nf.orthogonalize(torch.zeros(3, 0, device='cuda'))
    with pytest.raises(TypeError):
        nf.orthogonalize(g.double())
    with pytest.raises(NotImplementedError):
        nf.orthogonalize(g.requires_grad_())
    with torch.no_grad():
        assert not nf.orthogonalize(g).any()
    p, q, m = (torch.zeros(4, 6, device='cuda') for _ in range(3))
    for args in (([p], [q[:3]], [m]), ([p, p], [q, q], [m, m.clone()]), ([p], [q], [q]), ([p], [p], [m]),
                 ([p.t()], [q.t()], [m.t()]), ([p[0]], [q[0]], [m[0]])):
        with pytest.raises(ValueError):
            nf.muon_update(*args, lr=0.1)
    with pytest.raises(TypeError):
        nf.muon_update([p.double()], [q.double()], [m.double()], lr=0.1)
    assert not p.any() and not m.any()


def muon_oracle(p, g, m, lr, momentum=0.95, nesterov=True, weight_decay=0., steps=5, eps=1e-7):
    """(param, momentum, tolerance of the param) in float64."""
    m = momentum * m.double() + g.double()
    u = g.double() + momentum * m if nesterov else m
    o = iterate(u, steps, eps)
    rate = lr * math.sqrt(max(1, p.shape[0] / p.shape[1]))
    # (three roundings of the parameter: the factor 1 - lr wd, the product with it and the sum)
    tol = rate * tolerance(u, o, torch.float32, steps, eps, blocks=True) + 3 * 2.0 ** -24 * (norm(p) + rate * norm(o))
    return (1 - lr * weight_decay) * p.double() - rate * o, m, tol


def check_muon(shapes, seed, **kw):
    gen = torch.Generator().manual_seed(seed)
    ps = [0.1 * torch.randn(*s, generator=gen).cuda() for s in shapes]
    gs = [gradients(s, seed + i) for i, s in enumerate(shapes)]
    ms = [gradients(s, seed + 100 + i, 1e-2) for i, s in enumerate(shapes)]
    want = [muon_oracle(p, g, m, **kw) for p, g, m in zip(ps, gs, ms)]
    versions = [t._version for t in ps + ms]
    keep = [g.clone() for g in gs]
    nf.muon_update(ps, gs, ms, **kw)
    assert all(t._version > v for t, v in zip(ps + ms, versions))
    for p, g, m, k, (wp, wm, tol) in zip(ps, gs, ms, keep, want):
        assert torch.equal(g, k)
        assert bool((norm(p.double() - wp) <= tol).all()), p.shape
        assert bool(((m.double() - wm).abs() <= 2.0 ** -23 * (wm.abs() + g.double().abs())).all()), p.shape


@pytest.mark.gpu
@pytest.mark.parametrize('kw', [dict(lr=0.02), dict(lr=0.1, nesterov=False, weight_decay=0.3),
                                dict(lr=0.0, momentum=0.0), dict(lr=0.5, steps=2, eps=1e-2)], ids=str)
def test_muon_update(kw):
    check_muon([(64, 32), (128, 128), (32, 64), (64, 32), (1, 1), (300, 20), (128, 128), (700, 30), (200, 90)], 9, **kw)


@pytest.mark.gpu
def test_muon_update_of_many_matrices_and_shapes():
    """More matrices (48) and shapes (8) than one sequence of launches takes."""
    check_muon([(8 + i % 11, 12) for i in range(60)], 3, lr=0.05)
    check_muon([(5, 7)] * 50, 4, lr=0.05)


@pytest.mark.gpu
def test_muon_update_of_long_and_short_matrices():
    """One shape's products in parts, the others' whole, in the same launches."""
    check_muon([(512, 300), (6000, 510), (512, 512), (90, 100), (20, 30), (512, 512)], 5, lr=0.02)


@pytest.mark.gpu
def test_muon_grads_of_other_layouts_and_empty_matrices():
    p, g, m = torch.randn(30, 20).cuda(), gradients((20, 30), 1).t(), torch.zeros(30, 20).cuda()
    want, wm, tol = muon_oracle(p, g, m, 0.1)
    e = torch.zeros(0, 5, device='cuda')
    nf.muon_update([e, p], [e.clone(), g], [e.clone(), m], lr=0.1)
    assert bool((norm(p.double() - want) <= tol).all()) and bool(((m - wm).abs() <= 2.0 ** -23 * wm.abs()).all())


@pytest.mark.gpu
def test_streams():
    g = gradients((4, 300, 200), 8)
    h = gradients((2, 100, 450), 9)
    want, other = nf.orthogonalize(g), nf.orthogonalize(h)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(3):                                  # two calls at work at once, each with a workspace of its own
        with torch.cuda.stream(side):
            a = nf.orthogonalize(g)
        got.append((a, nf.orthogonalize(h)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) and torch.equal(b, other) for a, b in got)


@pytest.mark.gpu
def test_captured_update():
    """The whole step recorded into a graph and replayed, with eager work between the replays."""
    shapes = [(70, 40), (64, 64), (40, 90)]
    ps, ms = ([torch.zeros(s, device='cuda') for s in shapes] for _ in range(2))
    gs = [gradients(s, 1) for s in shapes]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        nf.muon_update(ps, gs, ms, lr=0.1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nf.muon_update(ps, gs, ms, lr=0.1)
    eager = [[t.clone() for t in ts] for ts in (ps, ms)]
    for seed in range(4):
        for g, s in zip(gs, shapes):
            g.copy_(gradients(s, seed + 20))
        graph.replay()
        torch.cuda.synchronize()
        nf.muon_update(eager[0], gs, eager[1], lr=0.1)
        for a, b in zip(ps + ms, eager[0] + eager[1]):
            assert torch.equal(a, b), seed


def small_flow(seed=0):
    torch.manual_seed(seed)
    mask = torch.arange(6) % 2
    layers = [nf.PiecewiseRationalQuadraticCouplingTransform(
        m, lambda i, o: nf.ResidualNet(i, o, 32, use_layer_norm=True), num_bins=8, tails='linear', tail_bound=3.)
        for m in (mask, 1 - mask)]
    layers.append(nf.MaskedPiecewiseRationalQuadraticAutoregressiveTransform(6, 24, num_bins=8, tails='linear', tail_bound=3.))
    return nf.BaseNeuralSplineFlow(nf.CompositeTransform(layers), nf.StandardNormal([6])).cuda()


def optimizers(flow):
    mats = [p for p in flow.parameters() if p.dim() == 2]
    return nf.Muon(mats, lr=0.02, weight_decay=0.01), \
        torch.optim.Adam([p for p in flow.parameters() if p.dim() != 2], lr=1e-2)


@pytest.mark.gpu
def test_training_run_with_layer_norm_and_muon():
    """A flow of layer-normalised coupling layers and a masked layer, trained by Muon and Adam: every Muon step is the
    formula's on the gradients that the backward kernels left, the layers see the new weights at once, and a run resumed
    from state dicts goes on with the same bits."""
    flow = small_flow()
    muon, adam = optimizers(flow)
    x = torch.randn(256, 6, generator=torch.Generator().manual_seed(1)).cuda()
    mats = muon.param_groups[0]['params']
    saved = None
    for step in range(4):
        if step == 2:
            saved = ({k: v.clone() for k, v in flow.state_dict().items()}, muon.state_dict(), adam.state_dict())
            saved = (saved[0], torch.utils._pytree.tree_map(lambda t: t.clone() if torch.is_tensor(t) else t, saved[1:]))
        muon.zero_grad()
        adam.zero_grad()
        loss = -flow.log_prob(x).mean()
        loss.backward()
        old = [p.detach().clone() for p in mats]
        buf = [muon.state[p].get('momentum_buffer', torch.zeros_like(p)).clone() for p in mats]
        muon.step()
        adam.step()
        for p, q, m in zip(mats, old, buf):
            want, _, tol = muon_oracle(q, p.grad, m, lr=0.02, weight_decay=0.01)
            assert p.grad.isfinite().all() and bool((norm(p.detach().double() - want) <= tol).all())
        with torch.no_grad():
            fresh = small_flow(5)
            fresh.load_state_dict(flow.state_dict())
            assert torch.equal(flow.log_prob(x), fresh.log_prob(x))         # no stale weight pack
    other = small_flow(7)
    other.load_state_dict(saved[0])
    muon2, adam2 = optimizers(other)
    muon2.load_state_dict(saved[1][0])
    adam2.load_state_dict(saved[1][1])
    for _ in range(2):
        muon2.zero_grad()
        adam2.zero_grad()
        (-other.log_prob(x).mean()).backward()
        muon2.step()
        adam2.step()
    # (the parameters of the two runs: equal up to the order of the weight-gradient atomics of the other kernels)
    for p, q in zip(flow.parameters(), other.parameters()):
        assert (p - q).abs().max().item() < 1e-3


@pytest.mark.gpu
def test_gradient_synchronizer_buckets_feed_the_step():
    """Gradients that are views into flat buckets (any 4-byte alignment) are read where they are."""
    flow = small_flow()
    sync = nf.parallel.GradientSynchronizer(flow.parameters())
    x = torch.randn(64, 6, generator=torch.Generator().manual_seed(2)).cuda()
    muon, _ = optimizers(flow)
    sync.zero_grad()
    (-flow.log_prob(x).mean()).backward()
    sync.finish()
    mats = muon.param_groups[0]['params']
    want = [muon_oracle(p.detach(), p.grad, torch.zeros_like(p), lr=0.02, weight_decay=0.01) for p in mats]
    muon.step()
    for p, (w, _, tol) in zip(mats, want):
        assert bool((norm(p.detach().double() - w) <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize('kind', TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize('shape', [(20, 300), (70, 90), (96, 100), (150, 140), (80, 700), (256, 1024), (130, 6000), (2, 600, 9),
                                   (500, 1100)], ids=str)
def test_norms_far_below_eps(shape, kind):
    """|G| << eps leaves X0 = G / (|G| + eps) small throughout; the steps lift it by a each until it is not.  Nothing in that is
    less exact than elsewhere: the same tolerance, on every path, for the steps that stay small and for those that do not."""
    g = gradients(shape, 1).to(kind)
    size = norm(g).max().item()
    for ratio, steps in ((1.0, 5), (0.1, 5), (1e-2, 5), (1e-5, 5), (1e-9, 5), (1e-12, 5), (1e-25, 5), (1e-36, 2), (1e-4, 11), (1e-12, 26)):
        eps = size / ratio
        check(nf.orthogonalize(g, steps=steps, eps=eps), g, kind, steps=steps, eps=eps)


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(20, 300), (70, 90), (150, 140), (80, 700), (130, 6000)], ids=str)
def test_each_matrix_has_its_own_scale(shape):
    """One batch of norms around eps and from far above it to far below; and of zeros."""
    g = torch.stack([gradients(shape, i, s) for i, s in enumerate((1e-3, 1e-17, 1e-10, 0.0, 1e3))])
    out = nf.orthogonalize(g)
    check(out, g, torch.float32)
    assert not out[3].any()


@pytest.mark.gpu
@pytest.mark.parametrize('shapes', [[(20, 300), (70, 90), (96, 40)], [(150, 140), (20, 300), (70, 90)], [(80, 700), (64, 64)],
                                    [(256, 1024), (130, 6000)]], ids=str)
def test_muon_norms_far_below_eps(shapes):
    for eps in (1e-7, 1e2, 1e9):
        ps, ms = ([torch.zeros(s, device='cuda') for s in shapes] for _ in range(2))
        gs = [gradients(s, i) for i, s in enumerate(shapes)]
        want = [muon_oracle(p, g, m, 0.5, eps=eps) for p, g, m in zip(ps, gs, ms)]
        nf.muon_update(ps, gs, ms, lr=0.5, eps=eps)
        for p, (w, _, tol) in zip(ps, want):
            assert bool((norm(p.double() - w) <= tol).all()), (eps, p.shape)


@pytest.mark.gpu
@pytest.mark.parametrize('shape', [(20, 70), (20, 700), (40, 70), (130, 150), (70, 900)], ids=str)
def test_zeros_over_the_smallest_eps(shape):
    """0 / (0 + eps) = 0 where eps, its reciprocal or that one's square leave the range of float64; 0 / 0 is NaN."""
    g = torch.zeros(shape, device='cuda')
    for eps in (1e-7, 1e-160, 1e-300, 1e-310, 5e-324):
        assert torch.equal(nf.orthogonalize(g, eps=eps), g)
    assert nf.orthogonalize(g, eps=0.0).isnan().all()
    h = gradients(shape, 1)
    assert torch.equal(nf.orthogonalize(h, eps=5e-324), nf.orthogonalize(h, eps=0.0))


@pytest.mark.parametrize('elem', [0, 1])
@pytest.mark.parametrize('rows,cols,counts', [(33, 32544, (254, 255, 256, 257, 300)), (64, 27936, (300, 340, 341, 342, 400)),
                                              (300, 3000, range(1, 60)), (100, 3000, range(1, 700, 7)), (4096, 4096, (1, 2, 3, 4)),
                                              (2500, 700, range(1, 80)), (20, 9000, range(1, 9))])
def test_a_workspace_does_for_every_smaller_count(rows, cols, counts, elem):
    """More matrices are cut into fewer parts of their k loops, so what the parts take does not grow with the count; the answer
    has to, since a batch that is cut ends with a smaller part."""
    lib = nf._lib.load()
    need = [lib.nf_orthogonalize_workspace_bytes(n, rows, cols, elem) for n in counts]
    assert need[0] > 0 and all(a <= b for a, b in zip(need, need[1:]))


@pytest.mark.gpu
@pytest.mark.parametrize('shape,per', [((11, 300, 3000), 6), ((7, 130, 3000), 3), ((5, 20, 3000), 2), ((9, 100, 3000), 4)], ids=str)
def test_a_cut_batch_of_matrices_in_parts(shape, per, monkeypatch):
    """A shorter last part, whose k loops are cut into more parts than the others'."""
    g = gradients(shape, 6)
    monkeypatch.setattr(nf._lib, 'WORKSPACE_BYTES', per * nf._lib.load().nf_orthogonalize_workspace_bytes(1, *shape[1:], 0))
    check(nf.orthogonalize(g), g, torch.float32)


def plain_update(u, eps=1e-7):
    """The update in torch's fp32 products, step by step."""
    x = u if u.shape[0] <= u.shape[1] else u.T.contiguous()
    x = x / (x.norm() + eps)
    for _ in range(5):
        s = x @ x.T
        x = A * x + (B * s + C * s @ s) @ x
    return x if u.shape[0] <= u.shape[1] else x.T


@pytest.mark.gpu
@pytest.mark.parametrize('decades', [0, 2, 4])
@pytest.mark.parametrize('shapes', [[(200, 2000)], [(1000, 384)], [(64, 128)], [(128, 700), (128, 128)],
                                    [(512, 784), (512, 512), (512, 512), (4000, 512)], [(128, 64), (128, 128), (1472, 128)]], ids=str)
def test_muon_keeps_the_digits_of_single_steps(shapes, decades):
    """The Muon step of parameters that start at zero is the update alone: as exact as a float32 result of nf.orthogonalize, by
    the measure of test_wide_fp32_keeps_the_digits_of_single_steps (torch's fp32 products, half as much again), over the step's
    matrices together.

    That measure alone does not hold for equal singular values (decades = 0): S is then a multiple of the identity, K squares
    of one sign, which the kernels sum in 3 K / 16 fp32 additions one after the other - at K = 2000 an error of
    0.58 * 2^-24 sqrt(3 * 2000 / 16 + 16) = 6.8e-7 of S, by the model above - and a library that adds its K in several sums
    that it joins does not have it (its whole error there is 3.4e-7).  So there `spread`, what the model's roundings of single steps
    come to, is added."""
    gen = torch.Generator().manual_seed(8)
    gs = []
    for m, n in shapes:
        k = min(m, n)
        u, v = (torch.linalg.qr(torch.randn(d, k, generator=gen, dtype=torch.float64))[0] for d in (m, n))
        gs.append(((u * 10 ** (-decades * torch.arange(k) / k)) @ v.T).float().cuda())
    ps, ms = ([torch.zeros(s, device='cuda') for s in shapes] for _ in range(2))
    nf.muon_update(ps, gs, ms, lr=1.0, momentum=0.0)
    sums = [0.0, 0.0, 0.0]
    for p, g in zip(ps, gs):
        want, rate = iterate(g), math.sqrt(max(1, g.shape[0] / g.shape[1]))
        model = iterate(g, gen=torch.Generator(device='cuda').manual_seed(77))
        for i, e in enumerate((-p - rate * want, rate * (plain_update(g) - want), rate * (model - want))):
            sums[i] += norm(e).item() ** 2
    ours, plain, spread = (math.sqrt(v) for v in sums)
    assert ours <= 1.5 * plain + (spread if decades == 0 else 0), (ours, plain, spread)


@pytest.mark.gpu
def test_forward_mode_is_refused():
    from torch.autograd import forward_ad
    g = gradients((6, 9), 1)
    p, m = torch.zeros_like(g), torch.zeros_like(g)
    want = nf.orthogonalize(g)
    with forward_ad.dual_level():
        assert torch.equal(nf.orthogonalize(g), want)
        dual = forward_ad.make_dual(g, torch.ones_like(g))
        with pytest.raises(NotImplementedError, match='tangent'):
            nf.orthogonalize(dual)
        for args in (([p], [dual], [m]), ([dual], [p], [m]), ([p], [m], [dual])):
            with pytest.raises(NotImplementedError, match='tangent'):
                nf.muon_update(*args, lr=0.1)
    assert not p.any() and not m.any()


@pytest.mark.gpu
def test_captured_optimizer_step():
    """The first step makes the momentum buffers: recorded into a graph they would be cleared at every replay, so that is refused.
    Later steps replay with the same bits as eager ones, the momentum carried on."""
    ps = [torch.nn.Parameter(gradients(s, 3, 0.1)) for s in ((70, 40), (20, 30))]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt, eager = nf.Muon(ps, lr=0.1), nf.Muon(qs, lr=0.1)
    for i, (p, q) in enumerate(zip(ps, qs)):
        p.grad = gradients(p.shape, i)
        q.grad = p.grad.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match='one step before'):
            opt.step()
        kept = ps[0].grad + 1
    graph.replay()
    assert torch.equal(kept, ps[0].grad + 1) and all(torch.equal(p, q) for p, q in zip(ps, qs))
    opt.step()
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for seed in range(4):
        for i, (p, q) in enumerate(zip(ps, qs)):
            p.grad.copy_(gradients(p.shape, 10 * seed + i))
            q.grad.copy_(p.grad)
        graph.replay()
        torch.cuda.synchronize()
        eager.step()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), seed


@pytest.mark.gpu
@pytest.mark.parametrize('kind', [torch.float32, torch.bfloat16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize('shape', [(3, 2050, 2200), (3, 2200, 2050), (2, 2100, 3000)], ids=str)
def test_the_largest_tiles_at_their_ends(shape, kind):
    """Batches that fill the device with tiles of 8 x 4 cells, which cross the matrix's end in both directions."""
    g = gradients(shape, 4).to(kind)
    out = nf.orthogonalize(g)
    check(out, g, kind)
    assert torch.equal(nf.orthogonalize(g), out)


@pytest.mark.gpu
@pytest.mark.parametrize('shapes', [[(2100, 2300)], [(2300, 2100)], [(2051, 2303)], [(2303, 2051)], [(2060, 2300), (2303, 2100)]],
                         ids=str)
def test_muon_with_the_largest_tiles(shapes):
    """Parameters in rows of whole 16 bytes and not, as they are and transposed, of one shape and of two."""
    check_muon(shapes * 2 + shapes[:1], 6, lr=0.02, weight_decay=0.1)


@pytest.mark.gpu
def test_largest_tiles_far_below_eps():
    g = gradients((3, 2050, 2200), 4)
    for ratio in (1e-3, 1e-12):
        check(nf.orthogonalize(g, eps=norm(g).max().item() / ratio), g, torch.float32, eps=norm(g).max().item() / ratio)
