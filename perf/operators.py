"""Cases of the optimizer operators: Newton-Schulz orthogonalisation of a ragged set of matrices (`orthogonalize`), the Muon
step built on it (`muon_step`) and the AdamW step of the parameters that are not matrices (`adamw_step`).

Matrix sizes are those of the shipped detector configurations (conv weights as output channels x taps * input channels, the
normalizing flows' linear layers, the predictors) or generic; `shapes` is "COUNTxROWSxCOLS;..." in the order of the storage.
"""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
NS_EPS = 1e-7

# every weight matrix of the two-stage MSPN2 + FPN + DASHead detector (configs/das/exp_panoptic.py), grouped by shape
DETECTOR = ('28x256x2304;6x512x4608;6x2048x512;2x2048x1024;4x512x2048;1x2048x2048;13x1024x256;12x256x1024;8x128x1152;'
            '2x1024x512;2x512x1024;2x256x2048;1x1024x1024;14x256x256;8x512x128;4x256x512;1x2048x256;3x512x256;6x128x512;'
            '1x512x512;4x27x2304;6x64x576;50x64x64;1x64x2304;8x256x64;5x64x256;2x128x256;5x45x256;1x120x256;1x64x147;'
            '24x64x3;24x3x64;24x64x2;24x2x64;2x1x256;1x2x256;1x1x64')


def listed():
    orth = dict(op='orthogonalize')
    muon = dict(op='muon', lr=2e-3, momentum=0.95, weight_decay=0.01, nesterov=True, max_norm=0.0)
    adam = dict(op='adamw', lr=2e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, max_norm=0.0)
    return [
        # one square linear layer of a flow: the smallest call, all latency
        dict(orth, name='orth 64x64', shapes='1x64x64', dtype='f32'),
        # one 3x3 conv weight, 256 -> 256 channels, from bf16 gradients: few tiles, a long inner axis
        dict(orth, name='orth 256x2304', shapes='1x256x2304', dtype='bf16'),
        # odd and ragged: predictor rows, the stem's 147 columns, a single row, a tall matrix, sizes that are multiples of nothing
        dict(orth, name='orth ragged', shapes='3x45x256;2x27x2304;1x64x147;2x1x256;1x333x77;2x129x1023;1x700x513', dtype='f32'),
        # a stack of wide projections: the largest products
        dict(orth, name='orth 4x 2048x8192', shapes='4x2048x8192', dtype='bf16'),
        # the flows' and predictors' matrices alone: many tiny ones
        dict(muon, name='muon small set', shapes='50x64x64;24x64x3;24x3x64;24x64x2;24x2x64;5x45x256;2x1x256'),
        # the 1x1 and 3x3 weights of one bottleneck of 512 channels
        dict(muon, name='muon bottleneck', shapes='1x512x2048;1x512x4608;1x2048x512'),
        # the whole two-stage detector with global-norm clipping: a training step's update
        dict(muon, name='muon detector', shapes=DETECTOR, max_norm=35.0),
        # two large square weights, plain (heavy-ball) momentum
        dict(muon, name='muon 2x 4096x4096', shapes='2x4096x4096', nesterov=False, momentum=0.9),
        # a vector of odd length: latency
        dict(adam, name='adamw 4099', n=4099, step=1),
        # what is left of the detector beside its matrices (BatchNorm / GroupNorm affines, biases, scales), clipped
        dict(adam, name='adamw 148754', n=148754, step=1000, max_norm=35.0),
        # a mid-size buffer
        dict(adam, name='adamw 5M', n=5_000_003, step=20),
        # a whole detector trained with AdamW
        dict(adam, name='adamw 66M', n=66_375_444, step=5000, weight_decay=0.05),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['orthogonalize', 'muon', 'adamw'])
    if op == 'adamw':
        return dict(op=op, n=_log_int(rng, 1, 60_000_000), step=_log_int(rng, 1, 100_000), lr=10 ** rng.uniform(-4, -2.5),
                    beta1=rng.choice([0.9, 0.95]), beta2=rng.choice([0.95, 0.99, 0.999]), eps=1e-8,
                    weight_decay=rng.choice([0.0, 0.01, 0.1]), max_norm=rng.choice([0.0, 1.0, 35.0]))
    while True:
        shapes, cost = [], 0.0
        for _ in range(rng.choice([1, 1, 2, 3, 5])):
            k, r, c = _log_int(rng, 1, 12), _log_int(rng, 1, 4096), _log_int(rng, 1, 8192)
            if rng.random() < 0.5:       # channel counts are multiples of 16 more often than not
                r, c = -(-r // 16) * 16, -(-c // 16) * 16
            shapes.append((k, r, c))
            m, n = min(r, c), max(r, c)
            cost += k * (15.0 * m * m * n + 5.0 * m ** 3)
        if cost <= 6e11 and sum(k * r * c for k, r, c in shapes) <= 60_000_000:
            break
    case = dict(op=op, shapes=';'.join('%dx%dx%d' % s for s in shapes))
    if op == 'orthogonalize':
        return dict(case, dtype=rng.choice(['f32', 'bf16']))
    return dict(case, lr=10 ** rng.uniform(-4, -2.5), momentum=rng.choice([0.9, 0.95, 0.98]), nesterov=rng.random() < 0.7,
                weight_decay=rng.choice([0.0, 0.01, 0.1]), max_norm=rng.choice([0.0, 1.0, 35.0]))


def _shapes(case):
    return [tuple(int(v) for v in s.split('x')) for s in case['shapes'].split(';')]


def _gradient(gen, k, r, c):
    """What a layer's weight gradient is made of: a sum over pixels of output gradients (channels of very different size)
    times rectified features that share a common part."""
    dev = 'cuda'
    pix = 2 * max(r, c) + 64
    x = torch.randn(pix, c, generator=gen, device=dev)
    x += torch.randn(pix, 1, generator=gen, device=dev)
    x = x.relu_()
    out = torch.empty(k, r, c, device=dev)
    for i in range(k):
        d = torch.randn(pix, r, generator=gen, device=dev) * torch.exp(torch.randn(r, generator=gen, device=dev))
        torch.mm(d.t(), x, out=out[i])
    return out.mul_(1e-3 / math.sqrt(pix))


def prepare(case, seed):
    gen = torch.Generator('cuda').manual_seed(seed)
    state = dict(case)
    if case['op'] == 'adamw':
        n = case['n']
        g = torch.randn(n, generator=gen, device='cuda') * torch.exp(2 * torch.randn(n, generator=gen, device='cuda')) * 1e-3
        t = case['step']
        b1, b2 = case['beta1'], case['beta2']
        m = torch.zeros_like(g) if t == 1 else 0.3 * torch.randn(n, generator=gen, device='cuda') * g.abs()
        v = torch.zeros_like(g) if t == 1 else (1 - b2 ** t) * torch.rand(n, generator=gen, device='cuda') * 2 * g * g
        p = 0.05 * torch.randn(n, generator=gen, device='cuda')
        state.update(p=p, g=g, m=m * (1 - b1 ** t), v=v)
        return state
    shapes = _shapes(case)
    if case['op'] == 'orthogonalize':
        dt = torch.float32 if case['dtype'] == 'f32' else torch.bfloat16
        state['mats'] = [_gradient(gen, *s).to(dt) for s in shapes]
        if own:
            from das_amd import train_ops
            state['plan'] = train_ops.NewtonSchulzPlan(shapes, 'cuda', steps=STEPS, coefficients=COEFFICIENTS, eps=NS_EPS)
        return state
    total = sum(k * r * c for k, r, c in shapes)
    g, m, p = (torch.empty(total, device='cuda') for _ in range(3))
    o = 0
    for k, r, c in shapes:       # matrices of one flat buffer, back to back
        e = o + k * r * c
        g[o:e] = _gradient(gen, k, r, c).view(-1)
        m[o:e] = 0.5 * (g[o:e] + _gradient(gen, k, r, c).view(-1))
        p[o:e] = torch.randn(k * r * c, generator=gen, device='cuda') * math.sqrt(2.0 / c)
        o = e
    state.update(p=p, g=g, m=m)
    if own:
        from das_amd import train_ops
        state['plan'] = train_ops.NewtonSchulzPlan(shapes, 'cuda', steps=STEPS, coefficients=COEFFICIENTS, eps=NS_EPS)
    return state


def _newton_schulz(u):
    """Plain form: a stack of equal matrices (k, r, c) in float32."""
    a, b, c = COEFFICIENTS
    x = u / (torch.sqrt((u * u).sum((1, 2), keepdim=True)) + NS_EPS)
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    for _ in range(STEPS):
        s = torch.matmul(x, x.transpose(1, 2))
        x = a * x + torch.matmul(b * s + c * torch.matmul(s, s), x)
    return x.transpose(1, 2) if tall else x


def _clip(g, max_norm):
    if max_norm <= 0:
        return g
    norm = torch.sqrt(g.double().square().sum())
    return g * torch.clamp(max_norm / (norm + 1e-6), max=1.0).float()


def run(state):
    if own:
        return _run_own(state)
    if state['op'] == 'orthogonalize':
        return [_newton_schulz(t.float()).to(torch.bfloat16) for t in state['mats']]
    p, g, m, lr, wd = state['p'], state['g'], state['m'], state['lr'], state['weight_decay']
    g = _clip(g, state['max_norm'])
    if state['op'] == 'adamw':
        v, b1, b2, t = state['v'], state['beta1'], state['beta2'], state['step']
        m.mul_(b1).add_(g, alpha=1 - b1)
        v.mul_(b2).add_(g * g, alpha=1 - b2)
        p.mul_(1 - lr * wd)
        p.sub_((m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + state['eps']) * lr)
        return {'p': p, 'm': m, 'v': v}
    mu = state['momentum']
    m.mul_(mu).add_(g, alpha=1 - mu)
    u = g * (1 - mu) + m * mu if state['nesterov'] else m
    p.mul_(1 - lr * wd)
    o = 0
    for k, r, c in _shapes(state):
        e = o + k * r * c
        x = _newton_schulz(u[o:e].view(k, r, c))
        p[o:e].view(k, r, c).sub_(x * (lr * math.sqrt(max(1.0, r / c))))
        o = e
    return {'p': p, 'm': m}


def _run_own(state):
    from das_amd import train_ops as T
    if state['op'] == 'orthogonalize':
        return T.orthogonalize(state['mats'], plan=state['plan'])
    p, g, m = state['p'], state['g'], state['m']
    sumsq = T.grad_sumsq(g) if state['max_norm'] > 0 else None
    if state['op'] == 'adamw':
        T.adamw_step(p, g, m, state['v'], lr=state['lr'], step=state['step'], beta1=state['beta1'], beta2=state['beta2'],
                     eps=state['eps'], weight_decay=state['weight_decay'], max_norm=state['max_norm'], grad_sumsq_t=sumsq)
        return {'p': p, 'm': m, 'v': state['v']}
    T.muon_step(p, g, m, state['plan'], lr=state['lr'], momentum=state['momentum'], weight_decay=state['weight_decay'],
                nesterov=state['nesterov'], max_norm=state['max_norm'], grad_sumsq_t=sumsq)
    return {'p': p, 'm': m}


def work(case):
    if case['op'] == 'adamw':
        return {'bytes': 28 * case['n'], 'flops': 16 * case['n']}
    size = flops = 0
    for k, r, c in _shapes(case):
        m, n = min(r, c), max(r, c)
        size += k * r * c
        # a symmetric product needs one half of its entries: X X^T (m m n), A A (m m m), then B X (2 m m n)
        flops += k * STEPS * (3 * m * m * n + m * m * m)
    each = 20 if case['op'] == 'muon' else (4 if case['dtype'] == 'f32' else 2) + 2
    return {'bytes': each * size, 'flops': flops}


def _polar64(u):
    """The odd polynomial s (a + b s^2 + c s^4), STEPS times, on one matrix in 64 bits: Horner on the smaller Gram matrix."""
    a, b, c = COEFFICIENTS
    x = u / (torch.linalg.vector_norm(u) + NS_EPS)
    wide = x.shape[0] <= x.shape[1]
    eye = torch.eye(min(x.shape), dtype=x.dtype, device=x.device)
    for _ in range(STEPS):
        gram = x @ x.mT if wide else x.mT @ x
        q = gram @ (c * gram + b * eye) + a * eye
        x = q @ x if wide else x @ q
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'orthogonalize':
        return [torch.stack([_polar64(t.double()) for t in stack]) for stack in s['mats']]
    p, g, m = s['p'].double(), s['g'].double(), s['m'].double()
    if case['max_norm'] > 0:
        total = float(torch.linalg.vector_norm(g))
        g = g * min(1.0, case['max_norm'] / (total + 1e-6))
    keep = 1.0 - case['lr'] * case['weight_decay']
    if case['op'] == 'adamw':
        b1, b2, t = case['beta1'], case['beta2'], case['step']
        m = torch.lerp(g, m, b1)
        v = torch.lerp(g.square(), s['v'].double(), b2)
        first, second = m / (1.0 - math.pow(b1, t)), v / (1.0 - math.pow(b2, t))
        return {'p': keep * p - case['lr'] * first / (second.sqrt() + case['eps']), 'm': m, 'v': v}
    m = torch.lerp(g, m, case['momentum'])
    u = torch.lerp(g, m, case['momentum']) if case['nesterov'] else m
    out, at = [], 0
    for k, r, c in _shapes(case):
        factor = case['lr'] * max(1.0, r / c) ** 0.5
        for _ in range(k):
            x = _polar64(u[at:at + r * c].view(r, c))
            out.append((keep * p[at:at + r * c].view(r, c) - factor * x).reshape(-1))
            at += r * c
    return {'p': torch.cat(out), 'm': m}
