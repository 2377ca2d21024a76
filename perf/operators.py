"""The training operators of a flow's conditioner networks, as they are measured: layer normalisation (inference and
training), the orthogonalisation of a matrix update and the whole Muon step over a flow's weight matrices.

`own` selects between the plain form (elementary torch operations in 32 bits) and this package's calls."""
import math

import torch

own = False

DEVICE = 'cuda'
TYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
EPS_NORM = 1e-5                                 # layer normalisation's epsilon
A, B, C = 3.4445, -4.7750, 2.0315               # the odd quintic a s + b s^3 + c s^5 of the orthogonalisation
STEPS, EPS_ORTH = 5, 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01


def listed():
    return [
        # a coupling conditioner (hidden 64) answering eight samples: latency
        {'name': 'norm_8x64', 'op': 'norm', 'rows': 8, 'features': 64, 'dtype': 'float32', 'pad': 0},
        # one inference pass of 131072 samples over hidden 512
        {'name': 'norm_131072x512', 'op': 'norm', 'rows': 131072, 'features': 512, 'dtype': 'float32', 'pad': 0},
        # a column slice of a wider half-precision activation: odd width, odd row stride
        {'name': 'norm_4099x1031_strided', 'op': 'norm', 'rows': 4099, 'features': 1031, 'dtype': 'float16', 'pad': 14},
        # training, a small batch of the coupling conditioner: forward, input gradient, weight and bias gradients
        {'name': 'norm_train_256x64', 'op': 'norm_train', 'rows': 256, 'features': 64, 'dtype': 'float32', 'pad': 0},
        # training at the batch of the training benchmark, hidden 512
        {'name': 'norm_train_32768x512', 'op': 'norm_train', 'rows': 32768, 'features': 512, 'dtype': 'float32',
         'pad': 0},
        # the largest: a wide conditioner kept in bf16
        {'name': 'norm_train_131072x2048', 'op': 'norm_train', 'rows': 131072, 'features': 2048, 'dtype': 'bfloat16',
         'pad': 0},
        # one small layer's update: latency
        {'name': 'orth_64x64', 'op': 'orth', 'batch': 1, 'rows': 64, 'cols': 64, 'dtype': 'float32'},
        # the hidden matrices of five autoregressive layers, two residual blocks each, as one batch
        {'name': 'orth_20x512x512', 'op': 'orth', 'batch': 20, 'rows': 512, 'cols': 512, 'dtype': 'float32'},
        # sizes that no tile divides, more rows than columns
        {'name': 'orth_3x1031x517', 'op': 'orth', 'batch': 3, 'rows': 1031, 'cols': 517, 'dtype': 'float16'},
        # a very wide conditioner's square matrix
        {'name': 'orth_4096x4096', 'op': 'orth', 'batch': 1, 'rows': 4096, 'cols': 4096, 'dtype': 'bfloat16'},
        # the step of a two-layer flow of 64 features, hidden 128
        {'name': 'muon_2x64x128', 'op': 'muon', 'features': 64, 'hidden': 128, 'blocks': 2, 'layers': 2, 'bins': 8,
         'nesterov': True},
        # the step of the headline model: five layers of 784 features, hidden 512, 8 bins
        {'name': 'muon_5x784x512', 'op': 'muon', 'features': 784, 'hidden': 512, 'blocks': 2, 'layers': 5, 'bins': 8,
         'nesterov': True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['norm', 'norm_train', 'orth', 'muon'])
    if op in ('norm', 'norm_train'):
        features = _log(rng, 1 if op == 'norm' else 8, 16384)
        return {'op': op, 'rows': _log(rng, 1, min(262144, 2 ** 28 // features)), 'features': features,
                'dtype': rng.choice(sorted(TYPES)), 'pad': rng.choice([0, 0, rng.randint(1, 64)])}
    if op == 'orth':
        rows, cols = _log(rng, 2, 4096), _log(rng, 2, 4096)
        return {'op': op, 'batch': _log(rng, 1, max(1, min(32, 2 ** 24 // (rows * cols)))), 'rows': rows, 'cols': cols,
                'dtype': rng.choice(sorted(TYPES))}
    return {'op': op, 'features': _log(rng, 4, 784), 'hidden': _log(rng, 8, 512), 'blocks': rng.randint(1, 2),
            'layers': rng.randint(1, 5), 'bins': rng.randint(2, 8), 'nesterov': rng.random() < 0.5}


def _gradient(gen, batch, rows, cols):
    """A weight gradient as a batch of samples leaves it: a few strong directions over a noise floor."""
    rank = max(1, min(rows, cols) // 8)
    u = torch.randn(batch, rows, rank, device=DEVICE, generator=gen)
    v = torch.randn(batch, rank, cols, device=DEVICE, generator=gen)
    return 1e-3 * ((u @ v) / math.sqrt(rank) + 0.1 * torch.randn(batch, rows, cols, device=DEVICE, generator=gen))


def _shapes(case):
    """(how often, rows, columns) of the weight matrices of a flow of autoregressive spline layers."""
    d, h, n = case['features'], case['hidden'], case['layers']
    return [(n, h, d), (n * 2 * case['blocks'], h, h), (n, d * (3 * case['bins'] - 1), h)]


def _masks(case):
    """The autoregressive masks of those three kinds of matrices: zero gradient where a weight is masked."""
    d, h = case['features'], case['hidden']
    inputs = torch.arange(1, d + 1, device=DEVICE)
    units = torch.arange(h, device=DEVICE) % max(1, d - 1) + min(1, d - 1)
    outputs = inputs.repeat_interleave(3 * case['bins'] - 1)
    return [units[:, None] >= inputs, units[:, None] >= units, outputs[:, None] > units]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    op = case['op']
    if op in ('norm', 'norm_train'):
        rows, n, kind = case['rows'], case['features'], TYPES[case['dtype']]
        wide = torch.randn(rows, n + case['pad'], device=DEVICE, generator=gen)
        wide = (1.5 * wide + torch.randn(rows, 1, device=DEVICE, generator=gen)).to(kind)
        state = {'op': op, 'x': wide[:, :n], 'weight': 1 + 0.2 * torch.randn(n, device=DEVICE, generator=gen),
                 'bias': 0.2 * torch.randn(n, device=DEVICE, generator=gen)}
        if op == 'norm_train':
            state['grad_y'] = torch.randn(rows, n, device=DEVICE, generator=gen).to(kind)
            for k in ('x', 'weight', 'bias'):
                state[k].requires_grad_()
        return state
    if op == 'orth':
        g = _gradient(gen, case['batch'], case['rows'], case['cols'])
        return {'op': op, 'matrices': g.to(TYPES[case['dtype']])}
    state = {'op': op, 'nesterov': case['nesterov'], 'params': [], 'grads': [], 'momenta': []}
    for (count, rows, cols), mask in zip(_shapes(case), _masks(case)):
        bound = 1 / math.sqrt(cols)
        state['params'] += list((2 * torch.rand(count, rows, cols, device=DEVICE, generator=gen) - 1) * bound)
        state['grads'] += [g.contiguous() for g in _gradient(gen, count, rows, cols) * mask]
        state['momenta'] += [g.contiguous() for g in 10 * _gradient(gen, count, rows, cols) * mask]
    return state


def _plain_norm(x, weight, bias):
    x = x.float()
    centred = x - x.mean(-1, keepdim=True)
    rstd = (centred.square().mean(-1, keepdim=True) + EPS_NORM).rsqrt()
    normed = centred * rstd
    return normed * weight + bias, normed, rstd


def _plain_orth(g):
    g = g.float()
    tall = g.shape[-2] > g.shape[-1]
    x = g.transpose(-1, -2) if tall else g
    x = x / (x.square().sum((-1, -2), keepdim=True).sqrt() + EPS_ORTH)
    for _ in range(STEPS):
        s = x @ x.transpose(-1, -2)
        x = A * x + (B * s + C * (s @ s)) @ x
    return x.transpose(-1, -2) if tall else x


@torch.no_grad()
def _plain(s):
    if s['op'] == 'norm':
        return _plain_norm(s['x'], s['weight'], s['bias'])[0].to(s['x'].dtype)
    if s['op'] == 'norm_train':
        y, normed, rstd = _plain_norm(s['x'], s['weight'], s['bias'])
        g = s['grad_y'].float()
        gw = g * s['weight']
        grad_x = rstd * (gw - gw.mean(-1, keepdim=True) - normed * (gw * normed).mean(-1, keepdim=True))
        return {'y': y.to(s['x'].dtype), 'grad_x': grad_x.to(s['x'].dtype), 'grad_weight': (g * normed).sum(0),
                'grad_bias': g.sum(0)}
    if s['op'] == 'orth':
        return _plain_orth(s['matrices']).to(s['matrices'].dtype)
    torch._foreach_mul_(s['momenta'], MOMENTUM)
    torch._foreach_add_(s['momenta'], s['grads'])
    updates = torch._foreach_add(s['grads'], s['momenta'], alpha=MOMENTUM) if s['nesterov'] else s['momenta']
    torch._foreach_mul_(s['params'], 1 - LR * DECAY)
    for shape in sorted({tuple(p.shape) for p in s['params']}):     # matrices of one shape go as one batch
        at = [i for i, p in enumerate(s['params']) if tuple(p.shape) == shape]
        o = _plain_orth(torch.stack([updates[i] for i in at]))
        torch._foreach_add_([s['params'][i] for i in at], list(o), alpha=-LR * math.sqrt(max(1, shape[0] / shape[1])))
    return {'params': s['params'], 'momenta': s['momenta']}


def run(s):
    if not own:
        return _plain(s)
    import normalizing_flows_amd as nf
    if s['op'] == 'norm':
        return nf.layer_norm(s['x'], s['weight'], s['bias'], eps=EPS_NORM)
    if s['op'] == 'norm_train':
        y = nf.layer_norm(s['x'], s['weight'], s['bias'], eps=EPS_NORM)
        grads = torch.autograd.grad(y, (s['x'], s['weight'], s['bias']), s['grad_y'])
        return {'y': y.detach(), 'grad_x': grads[0], 'grad_weight': grads[1], 'grad_bias': grads[2]}
    if s['op'] == 'orth':
        return nf.orthogonalize(s['matrices'], steps=STEPS, eps=EPS_ORTH)
    nf.muon_update(s['params'], s['grads'], s['momenta'], lr=LR, momentum=MOMENTUM, nesterov=s['nesterov'],
                   weight_decay=DECAY, steps=STEPS, eps=EPS_ORTH)
    return {'params': s['params'], 'momenta': s['momenta']}


def _orth_work(batch, rows, cols):
    """Products with a symmetric result (x x^T, s s) need half of it; (b s + c s s) x needs all."""
    m, n = min(rows, cols), max(rows, cols)
    return batch * STEPS * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    op = case['op']
    if op in ('norm', 'norm_train'):
        size = TYPES[case['dtype']].itemsize
        each = case['rows'] * case['features']
        passes, flops = (2, 8) if op == 'norm' else (4, 22)     # x, y; in training grad_y and grad_x too
        return {'bytes': passes * size * each + (8 if op == 'norm' else 16) * case['features'], 'flops': flops * each}
    if op == 'orth':
        return {'bytes': 2 * TYPES[case['dtype']].itemsize * case['batch'] * case['rows'] * case['cols'],
                'flops': _orth_work(case['batch'], case['rows'], case['cols'])}
    shapes = _shapes(case)
    # the parameter and the momentum read and written, the gradient read
    return {'bytes': sum(20 * k * r * c for k, r, c in shapes), 'flops': sum(_orth_work(*s) for s in shapes)}


def _exact_orth(g):
    """q(g g^T) g with the polynomial q carried along in the small Gram space, 64 bits."""
    g = g.double()
    if g.shape[-2] > g.shape[-1]:
        return _exact_orth(g.mT).mT
    x0 = g / (torch.linalg.matrix_norm(g)[..., None, None] + EPS_ORTH)
    one = torch.eye(g.shape[-2], dtype=torch.float64, device=g.device)
    gram, q = torch.matmul(x0, x0.mT), one
    for _ in range(STEPS):
        r = A * one + torch.matmul(B * one + C * gram, gram)
        q, gram = torch.matmul(r, q), torch.matmul(r, torch.matmul(gram, r))
    return torch.matmul(q, x0)


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if s['op'] in ('norm', 'norm_train'):
        x, w = s['x'].double(), s['weight'].double()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        scale = 1 / torch.sqrt(var + EPS_NORM)
        y = torch.addcmul(s['bias'].double(), (x - mean) * scale, w)
        if s['op'] == 'norm':
            return y
        # d/dx of the row's normalisation: the gradient without its part along (1, ..., 1) and along x - mean
        gy, n = s['grad_y'].double(), x.shape[1]
        u = gy * w
        along = torch.sum(u * (x - mean), 1, keepdim=True) / (n * (var + EPS_NORM))
        return {'y': y, 'grad_x': scale * (u - u.sum(1, keepdim=True) / n - (x - mean) * along),
                'grad_weight': torch.einsum('ij,ij->j', gy, (x - mean) * scale), 'grad_bias': gy.sum(0)}
    if s['op'] == 'orth':
        return _exact_orth(s['matrices'])
    params, momenta = [], []
    for p, g, m in zip(s['params'], s['grads'], s['momenta']):
        m = MOMENTUM * m.double() + g.double()
        u = g.double() + MOMENTUM * m if s['nesterov'] else m
        rate = LR * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        params.append(p.double() - LR * DECAY * p.double() - rate * _exact_orth(u))
        momenta.append(m)
    return {'params': params, 'momenta': momenta}
