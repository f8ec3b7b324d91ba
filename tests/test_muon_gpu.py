"""Newton-Schulz orthogonalisation, the Muon step and the AdamW step against 64-bit evaluations of their formulas."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
COEF = (3.4445, -4.7750, 2.0315)
U16 = 2.0 ** -11     # half a step of f16
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def gradient(r, c, seed, k=None):
    """a sum over pixels of output gradients times rectified features, as a layer's weight gradient is"""
    gen = torch.Generator().manual_seed(seed)
    n = (k or 1)
    out = []
    for _ in range(n):
        pix = 2 * max(r, c) + 16
        d = torch.randn(pix, r, generator=gen) * torch.exp(torch.randn(r, generator=gen))
        out.append(d.t() @ (torch.randn(pix, c, generator=gen) + torch.randn(pix, 1, generator=gen)).relu())
    g = torch.stack(out).to(DEV)
    return g if k else g[0]


def norm2(x):
    g = (x @ x.T if x.shape[0] <= x.shape[1] else x.T @ x).cpu()
    return math.sqrt(max(0.0, float(torch.linalg.eigvalsh((g + g.T) / 2)[-1])))


def ns64(u, coef, eps=1e-7, pairs=False):
    """(result in f64, bound on the 2-norm of the kernels' error). The bounds follow the roundings to first order. An error of X grows by at
    most L = max |p'| over the singular values' range in a step (the derivative of an odd function of a matrix is bounded, in the
    2-norm over all entries, by its divided differences). f32 sums: K inner elements are at most 3 K / 32 + 5 additions one after the other.
    f16 operands: X, G and Z are rounded by U16 (2^-25 absolute below the normal range; X is stored times about sqrt(n)).
    Pairs of f16: 2^-22 a rounding and 2^-22 for the dropped product of the low parts; steps are taken on G in phases, and what
    G and Q lose meanwhile is followed through G' = Z G Z and Q' = Z Q."""
    x = u.double()
    x = x / (x.norm() + eps)
    if x.shape[0] > x.shape[1]:
        y, e = ns64(u.t(), coef, eps, pairs)
        return y.t(), e
    m, n = x.shape
    rnd = 2.0 ** -22 if pairs else U16
    tiny = 2.0 ** -25 * math.sqrt(m) * 2
    eye = torch.eye(m, dtype=torch.float64, device=x.device)

    def acc(k):
        return (3 * k / 32 + 5) * 2.0 ** -23 + (2.0 ** -22 if pairs else 0)

    err = 2 * rnd * float(x.norm()) + 2 * tiny
    k = 0
    while k < len(coef):
        x0, g = x, x @ x.T
        eg = (rnd + acc(n)) * float(x.norm()) ** 2 + 2.0 ** -25 * m
        q, eq, grow = eye, 0.0, 1.0
        while True:
            a, b, c = coef[k]
            top = norm2(x)
            s = torch.linspace(0, max(top, 1e-30) * 1.01, 2048, dtype=torch.float64)
            err *= float((a + 3 * b * s ** 2 + 5 * c * s ** 4).abs().max())
            g2 = top * top
            z = a * eye + b * g + c * (g @ g)
            ez = (abs(b) + 2 * abs(c) * g2) * eg + abs(c) * acc(m) * float(g.norm()) ** 2 + \
                (rnd + 2.0 ** -22) * (float(z.norm()) + abs(b) * float(g.norm())) + 2.0 ** -25 * m
            zn, r = norm2(z), z @ g
            eq = zn * eq + norm2(q) * ez + (rnd + acc(m)) * float(z.norm()) * norm2(q)
            er = zn * eg + g2 * ez + (rnd + acc(m)) * float(z.norm()) * g2 + 2.0 ** -25 * m
            eg = zn * er + norm2(r) * ez + (rnd + acc(m)) * float(r.norm()) * zn + 2.0 ** -25 * m
            q, x, g = z @ q, z @ x, r @ z
            grow *= max(abs(a), zn) ** 2
            k += 1
            if k == len(coef) or not pairs or grow > 256:
                break
        err += eq * norm2(x0) + (rnd + acc(m)) * norm2(q) * float(x0.norm()) + tiny
    return x, err


def check(got, u, coef, eps=1e-7, what=''):
    ref, err = ns64(u, coef, eps, pairs=got.dtype == torch.float32)
    d = float((got.double() - ref).norm())
    tol = 1.1 * err + HALF[got.dtype] * float(ref.norm())
    assert torch.isfinite(got).all(), what
    assert d <= tol, (what, d, tol, float(ref.norm()))


SHAPES = [(1, 1), (1, 64), (64, 1), (2, 3), (45, 256), (27, 2304), (64, 64), (33, 200), (256, 64), (64, 257), (64, 147), (65, 63), (63, 65), (128, 1152), (129, 1023),
          (257, 64), (16, 1856), (16, 1857), (32, 769), (48, 480), (9, 5000), (3000, 33), (2, 20000), (333, 77), (512, 128), (500, 513), (700, 513), (256, 2304)]


@pytest.mark.parametrize('out_dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('steps', [1, 2, 5])
@pytest.mark.parametrize('shape', SHAPES, ids=lambda s: '%dx%d' % s)
def test_orthogonalize_one_matrix(shape, steps, out_dtype):
    from das_amd import train_ops as T
    u = gradient(*shape, seed=shape[0] * 7 + shape[1])
    check(T.orthogonalize(u, steps=steps, out_dtype=out_dtype), u, [COEF] * steps)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('out_dtype', [torch.bfloat16, torch.float16, torch.float32])
def test_orthogonalize_set(dtype, out_dtype):
    """every matrix of a ragged set, and a second call gives the same bits"""
    from das_amd import train_ops as T
    mats = [gradient(r, c, 3 * r + c, k=k) for k, r, c in [(3, 45, 256), (1, 333, 77), (2, 64, 64), (1, 1, 256), (5, 64, 3), (1, 129, 640)]]
    mats = [(t * (1e-3 if dtype == torch.float16 else 1)).to(dtype) for t in mats]
    plan = T.NewtonSchulzPlan([tuple(t.shape) for t in mats], DEV)
    got = T.orthogonalize(mats, plan=plan, out_dtype=out_dtype)
    again = T.orthogonalize(mats, plan=plan, out_dtype=out_dtype)
    for t, y, z in zip(mats, got, again):
        assert y.shape == t.shape and y.dtype == out_dtype and torch.equal(y, z)
        for i in range(t.shape[0]):
            check(y[i], t[i], [COEF] * 5, what=tuple(t.shape))


def test_orthogonalize_strides_and_offsets():
    """rows and stacks of any stride, starts that no vector load could take, a transposed view"""
    from das_amd import train_ops as T
    base = gradient(131, 407, 5)
    view = base[1:120, 3:400]
    check(T.orthogonalize(view), view, [COEF] * 5)
    stack = gradient(60, 100, 6, k=5)[::2, 1:, 1:98]
    for i, y in enumerate(T.orthogonalize(stack)):
        check(y, stack[i], [COEF] * 5)
    half = base.bfloat16()[:, 1:]
    check(T.orthogonalize(half), half, [COEF] * 5)
    check(T.orthogonalize(base.t()), base.t(), [COEF] * 5)
    same = base[:1].expand(64, -1)       # a row stride of zero: rank one
    check(T.orthogonalize(same), same, [COEF] * 5)


@pytest.mark.parametrize('mag', [1e-30, 1e-12, 1e12, 1e30])
def test_orthogonalize_magnitudes(mag):
    from das_amd import train_ops as T
    u = gradient(96, 160, 9)
    u = u / u.norm() * mag
    check(T.orthogonalize(u, eps=0.0 if mag < 1 else 1e-7), u, [COEF] * 5, eps=0.0 if mag < 1 else 1e-7)


def test_orthogonalize_hard_spectra():
    """rank one, low rank, zeros, a single huge entry"""
    from das_amd import train_ops as T
    gen = torch.Generator().manual_seed(1)
    a = (torch.randn(96, 8, generator=gen) @ torch.randn(8, 300, generator=gen)).to(DEV)
    one = torch.outer(torch.randn(70, generator=gen), torch.randn(200, generator=gen)).to(DEV)
    for dt in (torch.bfloat16, torch.float32):
        check(T.orthogonalize(a, out_dtype=dt), a, [COEF] * 5)
        check(T.orthogonalize(one, out_dtype=dt), one, [COEF] * 5)
    assert not T.orthogonalize(torch.zeros(40, 70, device=DEV)).any()
    spike = 1e-6 * torch.randn(65, 130, generator=gen)
    spike[64, 129] = 1e6
    spike = spike.to(DEV)
    check(T.orthogonalize(spike), spike, [COEF] * 5)


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_orthogonalize_nonfinite_stays_in_its_matrix(bad):
    from das_amd import train_ops as T
    a, b, c = gradient(64, 100, 1), gradient(70, 100, 2), gradient(100, 70, 3)
    d, e = gradient(40, 60, 4), gradient(40, 60, 5)
    clean = T.orthogonalize([a, b, c, d, e])
    b, d = b.clone(), d.clone()
    b[69, 99] = d[39, 0] = bad
    got = T.orthogonalize([a, b, c, d, e])
    for i in (0, 2, 4):
        assert torch.equal(got[i], clean[i])
    assert torch.isnan(got[1]).all() and torch.isnan(got[3]).all()


def test_orthogonalize_other_polynomials_and_empty():
    from das_amd import train_ops as T
    u = gradient(80, 120, 4)
    cubic = (1.5, -0.5, 0.0)
    check(T.orthogonalize(u, steps=3, coefficients=cubic), u, [cubic] * 3)
    per_step = [(4.0, -6.0, 2.5), (3.0, -4.0, 1.8), (2.0, -1.5, 0.5)]
    check(T.orthogonalize(u, steps=3, coefficients=per_step), u, per_step)
    check(T.orthogonalize(u, steps=3, coefficients=per_step, out_dtype=torch.float32), u, per_step)
    check(T.orthogonalize(u, steps=12, coefficients=cubic, out_dtype=torch.float32), u, [cubic] * 12)
    assert T.orthogonalize([]) == []
    e = T.orthogonalize([torch.zeros(0, 5, device=DEV), u, torch.zeros(3, 4, 0, device=DEV)])
    assert e[0].shape == (0, 5) and e[2].shape == (3, 4, 0) and torch.equal(e[1], T.orthogonalize(u))
    assert T.orthogonalize(torch.zeros(0, 7, device=DEV)).shape == (0, 7)


def test_orthogonalize_many_tensors():
    """more source tensors than one launch takes by value"""
    from das_amd import train_ops as T
    mats = [gradient(3 + i % 7, 5 + i % 11, 100 + i) for i in range(150)]
    for t, y in zip(mats, T.orthogonalize(mats)):
        check(y, t, [COEF] * 5)


def test_orthogonalize_twenty_thousand_matrices():
    """tables of more than a megabyte beside few elements"""
    from das_amd import train_ops as T
    t = gradient(2, 3, 8, k=20000)
    plan = T.NewtonSchulzPlan([(20000, 2, 3)], DEV)
    assert plan._flat[0].table_bytes > (1 << 20) + t.numel() // 16
    y = T.orthogonalize(t, plan=plan)
    for i in (0, 1, 9999, 19999):
        check(y[i], t[i], [COEF] * 5, what=i)


def test_orthogonalize_large_tiles():
    """sets of enough tiles for the 128 x 128 form, ragged at its edges"""
    from das_amd import train_ops as T
    mats = [gradient(300, 411, 1, k=40), gradient(257, 130, 2, k=30), gradient(129, 1025, 3, k=20)]
    for dt in (torch.bfloat16, torch.float32):
        for t, y in zip(mats, T.orthogonalize(mats, out_dtype=dt)):
            for i in (0, 7, t.shape[0] - 1):
                check(y[i], t[i], [COEF] * 5, what=(tuple(t.shape), i))


@pytest.mark.parametrize('many', [False, True])     # True: launches long enough for the second stream
def test_mixed_set_from_threads_streams_and_a_graph(many):
    """a set of every class (one workgroup, slices, tiles): the same bits alone, from two host threads on streams of their own at once, back to
    back on one stream with its input overwritten in between, and replayed"""
    import threading
    from das_amd import train_ops as T
    mats = [gradient(64, 64, 1, k=3), gradient(30, 3000, 2, k=2), gradient(200, 333, 3, k=2), gradient(5000, 12, 4)] + [gradient(256, 200, 5, k=60)] * many
    plan = T.NewtonSchulzPlan([tuple(t.shape) for t in mats], DEV)
    for dt in (torch.bfloat16, torch.float32):
        want = T.orthogonalize(mats, plan=plan, out_dtype=dt)
        twice = [t * 2 for t in mats]
        want2 = T.orthogonalize(twice, plan=plan, out_dtype=dt)
        for t, y in zip(mats, want):
            for i in range(y.shape[0] if y.dim() == 3 else 1):
                check(y[i] if y.dim() == 3 else y, t[i] if y.dim() == 3 else t, [COEF] * 5)
        torch.cuda.synchronize()
        wrong = []

        def work(src, ref):
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                buf = [t.clone() for t in src]
                got = []
                for _ in range(20):
                    got.append(T.orthogonalize(buf, plan=plan, out_dtype=dt))
                    for b, t in zip(buf, src):      # (the call's own work is ordered before this)
                        b.zero_()
                        b.copy_(t)
            s.synchronize()
            wrong.extend(1 for g in got for a, b in zip(g, ref) if not torch.equal(a, b))
        ts = [threading.Thread(target=work, args=a) for a in ((mats, want), (twice, want2))]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
        assert not wrong
        static, g = [t.clone() for t in mats], torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = T.orthogonalize(static, plan=plan, out_dtype=dt)
        for src, ref in ((twice, want2), (mats, want), (twice, want2)):
            for a, b in zip(static, src):
                a.copy_(b)
            g.replay()
            eager = T.orthogonalize(src, plan=plan, out_dtype=dt)
            torch.cuda.synchronize()
            for a, b, c in zip(out, eager, ref):
                assert torch.equal(a, c) and torch.equal(b, c)


def test_plan_serves_two_streams_and_a_graph():
    from das_amd import train_ops as T
    u, v = gradient(256, 300, 1), gradient(256, 300, 2)
    plan = T.NewtonSchulzPlan([(256, 300)], DEV)
    want_u, want_v = T.orthogonalize([u], plan=plan)[0], T.orthogonalize([v], plan=plan)[0]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        with torch.cuda.stream(s1):
            a = T.orthogonalize([u], plan=plan)[0]
        with torch.cuda.stream(s2):
            b = T.orthogonalize([v], plan=plan)[0]
        got.append((a, b))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, want_u) and torch.equal(b, want_v)
    static, g1, g2 = u.clone(), torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = T.orthogonalize([static], plan=plan)[0]
    with torch.cuda.graph(g2):
        o2 = T.orthogonalize([static], plan=plan)[0]
    for t, want in ((v, want_v), (u, want_u), (v, want_v)):
        static.copy_(t)
        g1.replay()
        g2.replay()
        extra = T.orthogonalize([t], plan=plan)[0]
        torch.cuda.synchronize()
        assert torch.equal(o1, want) and torch.equal(o2, want) and torch.equal(extra, want)


def muon64(p, g, m, shapes, offsets, lr, momentum, wd, nesterov, lr_scale, coef):
    p, g, m = p.double().clone(), g.double(), m.double().clone()
    tol = torch.zeros_like(p)
    for (k, r, c), o in zip(shapes, offsets):
        for i in range(k):
            s = slice(o + i * r * c, o + (i + 1) * r * c)
            m[s] = momentum * m[s] + (1 - momentum) * g[s] * coef
            u = (1 - momentum) * g[s] * coef + momentum * m[s] if nesterov else m[s]
            x, err = ns64(u.view(r, c), [COEF] * 5, pairs=True)
            f = math.sqrt(max(1.0, r / c)) if lr_scale == 'original' else 0.2 * math.sqrt(max(r, c))
            p[s] = p[s] * (1 - lr * wd) - lr * f * x.reshape(-1)
            tol[s] = 1.1 * lr * f * err      # (2-norm over the matrix)
    return p, m, tol


@pytest.mark.parametrize('nesterov,lr_scale,clip', [(True, 'original', 0.0), (False, 'match_rms_adamw', 0.0), (True, 'original', 0.5)])
def test_muon_step(nesterov, lr_scale, clip):
    """two steps over a flat buffer with gaps and odd starts between the matrices; the gaps keep their bytes"""
    from das_amd import train_ops as T
    shapes, offsets = [(2, 64, 147), (1, 300, 70), (3, 64, 3), (1, 1, 256), (1, 128, 256)], []
    at = 5
    for i, (k, r, c) in enumerate(shapes):
        offsets.append(at)
        at += k * r * c + (3, 1, 64, 17, 9)[i]
    gen = torch.Generator().manual_seed(3)
    p, g, m = (torch.randn(at, generator=gen).to(DEV) * s for s in (0.1, 1e-2, 1e-2))
    inside = torch.zeros(at, dtype=torch.bool, device=DEV)
    for (k, r, c), o in zip(shapes, offsets):
        inside[o:o + k * r * c] = True
    p0, m0 = p.clone(), m.clone()
    plan = T.NewtonSchulzPlan(shapes, DEV, offsets=offsets)
    kw = dict(lr=0.02, momentum=0.9, weight_decay=0.1, nesterov=nesterov, lr_scale=lr_scale)
    for step in range(2):
        sumsq = T.grad_sumsq(g)
        norm = float(g.double().norm()) * 0.5
        coef = 0.5 * (min(1.0, clip / (norm + 1e-6)) if clip else 1.0)
        rp, rm, tol = muon64(p, g, m, shapes, offsets, kw['lr'], kw['momentum'], kw['weight_decay'], nesterov, lr_scale, coef)
        T.muon_step(p, g, m, plan, grad_scale=0.5, max_norm=clip, grad_sumsq_t=sumsq, **kw)
        # momentum: products and a sum in f32, the clip factor from a f32 sum of squares over n elements
        assert float((m.double() - rm)[inside].abs().max()) <= (8 + 32 * (clip > 0)) * 2.0 ** -24 * float(rm.abs().max() + g.abs().max())
        for (k, r, c), o in zip(shapes, offsets):
            for i in range(k):
                s = slice(o + i * r * c, o + (i + 1) * r * c)
                slack = 4 * 2.0 ** -24 * float(p[s].double().norm()) + (1e-4 if clip else 0) * float(tol[o])
                assert float((p[s].double() - rp[s]).norm()) <= float(tol[s][0]) + slack, (step, r, c)
        g = torch.randn(at, generator=gen).to(DEV) * 1e-2
    assert torch.equal(p[~inside], p0[~inside]) and torch.equal(m[~inside], m0[~inside])
    assert not torch.equal(p[inside], p0[inside])


@pytest.mark.parametrize('n', [1, 3, 4, 5, 255, 4099, 1 << 20, 3_000_001])
@pytest.mark.parametrize('step,clip', [(1, 0.0), (7, 1.0), (100000, 0.0)])
def test_adamw_step(n, step, clip):
    from das_amd import train_ops as T
    gen = torch.Generator().manual_seed(n + step)
    p, g = torch.randn(n, generator=gen).to(DEV), (torch.randn(n, generator=gen) * torch.exp(3 * torch.randn(n, generator=gen))).to(DEV) * 1e-3
    m = torch.zeros_like(p) if step == 1 else g * torch.rand(n, generator=gen).to(DEV)
    v = torch.zeros_like(p) if step == 1 else g * g * torch.rand(n, generator=gen).to(DEV) * (1 - 0.999 ** step)
    kw = dict(lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1)
    sumsq = T.grad_sumsq(g)
    coef = 0.25 * (min(1.0, clip / (float(g.double().norm()) * 0.25 + 1e-6)) if clip else 1.0)
    gd = g.double() * coef
    m64 = 0.9 * m.double() + 0.1 * gd
    v64 = 0.999 * v.double() + 0.001 * gd * gd
    upd = (m64 / (1 - 0.9 ** step)) / ((v64 / (1 - 0.999 ** step)).sqrt() + 1e-8)
    p64 = p.double() * (1 - 1e-2 * 0.1) - 1e-2 * upd
    mag = 0.9 * m.double().abs() + 0.1 * gd.abs()
    T.adamw_step(p, g, m, v, step=step, grad_scale=0.25, max_norm=clip, grad_sumsq_t=sumsq, **kw)
    u = 2.0 ** -24
    cl = 64 * u if clip else 0.0      # the f32 sum of squares (a tree of partial sums) under the clip factor
    assert ((m.double() - m64).abs() <= (6 * u + cl) * mag).all()
    assert ((v.double() - v64).abs() <= (8 * u + 2 * cl) * v64 + 2.0 ** -126).all()
    # m carries an absolute error of (6 u + cl) mag (its two terms may cancel), the quotient and the root a dozen roundings more
    lim = (4 * u) * p64.abs() + 1e-2 * ((16 * u + 2 * cl) * upd.abs() + (6 * u + cl) * (mag / (1 - 0.9 ** step)) /
                                        ((v64 / (1 - 0.999 ** step)).sqrt() + 1e-8)) + 4 * u * p.double().abs()
    assert ((p.double() - p64).abs() <= lim).all()


def test_adamw_unaligned_views_and_empty():
    from das_amd import train_ops as T
    base = [torch.randn(1031, device=DEV).abs() for _ in range(4)]
    a = [t.clone() for t in base]
    T.adamw_step(*[t[1:1030] for t in a], lr=1e-2, step=3)
    b = [t[1:1030].clone() for t in base]
    T.adamw_step(*b, lr=1e-2, step=3)
    for x, y, z in zip(a, b, base):
        assert torch.equal(x[1:1030], y) and x[0] == z[0] and x[1030] == z[1030]
    T.adamw_step(*[torch.empty(0, device=DEV) for _ in range(4)], lr=1e-2, step=1)


def test_nan_norm_and_nan_gradient():
    from das_amd import train_ops as T
    p, m, v = (torch.ones(64, device=DEV) for _ in range(3))
    g = torch.ones(64, device=DEV)
    g[5] = float('nan')
    T.adamw_step(p, g, m, v, lr=1e-2, step=1)
    assert torch.isnan(p[5]) and int(torch.isnan(p).sum()) == 1
    T.adamw_step(p, g, m, v, lr=1e-2, step=1, max_norm=1.0, grad_sumsq_t=T.grad_sumsq(g))
    assert torch.isnan(p).all()


def test_refusals():
    from das_amd import train_ops as T
    from das_amd._lib import DasHipError
    u = torch.ones(8, 8, device=DEV)
    f = torch.ones(64, device=DEV)
    plan = T.NewtonSchulzPlan([(8, 8)], DEV)
    for bad in (lambda: T.orthogonalize(u, out_dtype=torch.float64), lambda: T.orthogonalize(u.double()),
                lambda: T.orthogonalize([u, u.half()]), lambda: T.orthogonalize(u[0]), lambda: T.orthogonalize(u.cpu()),
                lambda: T.orthogonalize([u, u], plan=plan), lambda: T.orthogonalize(u, steps=0), lambda: T.orthogonalize(u, steps=17),
                lambda: T.orthogonalize(u, coefficients=(float('nan'), 0, 0)), lambda: T.orthogonalize(u, coefficients=(40., 0, 0)),
                lambda: T.orthogonalize(u, coefficients=[(1.5, -.5, 0)] * 2), lambda: T.orthogonalize(u, eps=-1.0),
                lambda: T.NewtonSchulzPlan([(8, 8), (8, 8)], DEV, offsets=[0, 63]), lambda: T.NewtonSchulzPlan([(8, 8)], DEV, offsets=[-1]),
                lambda: T.NewtonSchulzPlan([(8, 8)], DEV, offsets=[0, 64]), lambda: T.NewtonSchulzPlan([(8, 8)], 'cpu'),
                lambda: T.NewtonSchulzPlan([(8, -8)], DEV),
                lambda: T.orthogonalize([u], plan=T.NewtonSchulzPlan([(8, 8)], DEV, offsets=[0])),
                lambda: T.muon_step(f[:63], f[:63], f[:63], plan, lr=1e-2), lambda: T.muon_step(f, f, f[:60], plan, lr=1e-2),
                lambda: T.muon_step(f, f, f.half(), plan, lr=1e-2), lambda: T.muon_step(f, f, f, plan, lr=1e-2, lr_scale='x'),
                lambda: T.muon_step(f, f, f, plan, lr=1e-2, momentum=1.0), lambda: T.muon_step(f, f, f, plan, lr=-1.0),
                lambda: T.muon_step(f, f, f, plan, lr=1e-2, max_norm=1.0), lambda: T.adamw_step(f, f, f, f, lr=1e-2, step=0),
                lambda: T.adamw_step(f, f, f, f, lr=1e-2, step=1, beta1=1.0), lambda: T.adamw_step(f, f, f, f, lr=float('nan'), step=1),
                lambda: T.adamw_step(f, f, f, f, lr=1e-2, step=1, max_norm=1.0),
                lambda: T.adamw_step(f, f, f, f.cpu(), lr=1e-2, step=1), lambda: T.adamw_step(f[::2], f[::2], f[::2], f[::2], lr=1e-2, step=1)):
        with pytest.raises(DasHipError):
            bad()
    assert (f == 1).all() and (u == 1).all()


def test_overlap_is_refused_and_neighbours_are_not():
    from das_amd import train_ops as T
    from das_amd._lib import DasHipError
    whole = torch.ones(4 * 64, device=DEV)
    parts = whole.split(64)
    plan = T.NewtonSchulzPlan([(8, 8)], DEV)
    for bad in (lambda: T.muon_step(parts[0], parts[0], parts[1], plan, lr=1e-2), lambda: T.muon_step(parts[0], parts[1], whole[32:96], plan, lr=1e-2),
                lambda: T.adamw_step(parts[0], parts[1], parts[2], parts[2], lr=1e-2, step=1),
                lambda: T.adamw_step(parts[0], whole[127:191], parts[1], parts[3], lr=1e-2, step=1),
                lambda: T.orthogonalize(whole.view(16, 16), coefficients=())):
        with pytest.raises(DasHipError):
            bad()
    assert (whole == 1).all()
    T.adamw_step(*parts, lr=1e-2, step=1)
    T.muon_step(*parts[:3], plan, lr=1e-2)
    assert torch.isfinite(whole).all() and (whole[64:128] == 1).all()


# ------------------------------------------------------------------ the optimizers in a training run
def detector():
    from test_train_step_gpu import make
    return make('f32')


@pytest.mark.parametrize('kind', ['AdamW', 'Muon'])
def test_optimizer_steps_follow_the_formulas(kind):
    """Two training steps of a small detector: every parameter against the 64-bit formula applied to the gradients the step saw, clipping
    and the bias rules included; the flat storage's padding stays zero."""
    from das_amd.optim import build_optimizer
    model, data = detector()
    cfg = dict(optimizer=dict(type=kind, lr=0.01, weight_decay=0.1, paramwise_cfg=dict(bias_lr_mult=2., bias_decay_mult=0.)),
               optimizer_config=dict(grad_clip=dict(max_norm=35, norm_type=2)))
    if kind == 'Muon':
        cfg['optimizer'].update(momentum=0.9, adamw_lr=1e-3)
    opt = build_optimizer(model, cfg)
    names = dict(zip(opt._names, zip(opt._params, opt.slots)))
    m64 = {n: torch.zeros(sl.numel, dtype=torch.float64, device=DEV) for n, (p, sl) in names.items()}
    v64 = {n: torch.zeros(sl.numel, dtype=torch.float64, device=DEV) for n, (p, sl) in names.items()}
    p_err = {n: 0.0 for n in names}
    groups = {n: next(g for g in opt.groups if g['start'] <= sl.off < g['end']) for n, (p, sl) in names.items()}
    if kind == 'Muon':
        assert sum(g['key'] == 'matrix' for g in groups.values()) > 20
        assert groups['bbox_head.conv_cls.weight']['key'] == 'main' and groups['backbone.top.top.0.conv.weight']['key'] == 'matrix'
    u = 2.0 ** -24
    for step in (1, 2):
        opt.zero_grad()
        model.train_step(data, None)['loss'].backward()
        opt.all_reduce_grads()
        norm = float(opt.flat_g.double().norm())
        k = min(1.0, 35 / (norm + 1e-6))
        before, g0 = opt.flat_p.clone(), opt.flat_g.clone()
        opt.step(0.01)
        for n, (p, sl) in names.items():
            s, g = slice(sl.off, sl.off + sl.numel), groups[n]
            lr, wd = 0.01 * g['lr_mult'], g['wd']
            gd, pd, got = g0[s].double() * k, before[s].double(), opt.flat_p[s].double()
            clip = 2.0 ** -17       # (the f32 sum of squares over the whole gradient)
            if g['key'] == 'matrix':
                m64[n] = 0.9 * m64[n] + 0.1 * gd
                r, c = p.shape[0], p.numel() // p.shape[0]
                w = 0.1 * gd + 0.9 * m64[n]
                x, err = ns64(w.view(r, c), [COEF] * 5, pairs=True)
                f = math.sqrt(max(1.0, r / c))
                want = pd * (1 - lr * wd) - lr * f * x.reshape(-1)
                # the input itself carries the clip factor's and the momentum's rounding: a relative error of U's norm, times L^5 <= 3.4445^5
                lim = lr * f * (1.1 * err + 485 * 16 * u) + 4 * u * float(pd.norm())
                assert float((got - want).norm()) <= lim, (n, step)
            else:
                m64[n] = 0.9 * m64[n] + 0.1 * gd
                v64[n] = 0.999 * v64[n] + 0.001 * gd * gd
                den = (v64[n] / (1 - 0.999 ** step)).sqrt() + 1e-8
                upd = (m64[n] / (1 - 0.9 ** step)) / den
                want = pd * (1 - lr * wd) - lr * upd
                # moments carry `clip` relative errors of their terms (|m| terms up to 2 |g| / den); the division and the root a few u
                lim = 8 * u * pd.abs() + lr * (64 * u + 4 * clip) * (upd.abs() + 2 * gd.abs() / den + 1)
                assert ((got - want).abs() <= lim).all(), (n, step)
        for n, (p, sl) in names.items():
            assert not opt.flat_p[sl.off + sl.numel:sl.off + sl.span].any()
    assert all(torch.isfinite(p).all() for p in model.parameters())


@pytest.mark.parametrize('kind', ['AdamW', 'Muon'])
def test_optimizer_resumes_bit_for_bit(kind):
    """state dict -> a fresh optimizer: same state, and the next step from the same parameters and gradients gives the same bits"""
    from das_amd.optim import build_optimizer, train_iteration
    cfg = dict(type=kind, lr=2e-3, weight_decay=0.01)
    model, data = detector()
    opt = build_optimizer(model, cfg)
    for _ in range(2):
        train_iteration(model, opt, data, 2e-3)
    other, _ = detector()
    other.load_state_dict(model.state_dict())
    opt2 = build_optimizer(other, cfg)
    opt2.load_state_dict(opt.state_dict())
    assert opt2.steps == 2 and torch.equal(opt2.flat_m, opt.flat_m) and torch.equal(opt2.flat_v, opt.flat_v)
    assert torch.equal(opt2.flat_p, opt.flat_p)
    opt2.flat_g.copy_(opt.flat_g)
    opt.step()
    opt2.step()
    assert torch.equal(opt2.flat_p, opt.flat_p) and torch.equal(opt2.flat_m, opt.flat_m)
    assert torch.isfinite(opt.flat_p).all()


def test_optimizer_refuses_capture():
    from das_amd.optim import FlatAdamW
    net = torch.nn.Linear(16, 16).to(DEV)
    opt = FlatAdamW(net, lr=1e-3)
    before = opt.flat_p.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        scratch = torch.zeros(4, device=DEV)
        with pytest.raises(RuntimeError):
            opt.step()
    assert opt.steps == 0 and torch.equal(opt.flat_p, before) and scratch.numel() == 4
    opt.step()
    assert opt.steps == 1


def test_steps_replay_in_a_graph():
    """the functional steps captured, with their fixed scalars: every replay equals the eager call, with eager work in between"""
    from das_amd import train_ops as T
    shapes = [(2, 130, 200), (3, 20, 30)]
    n = sum(k * r * c for k, r, c in shapes)
    gen = torch.Generator().manual_seed(0)
    p, g, m, v = (torch.randn(n, generator=gen).to(DEV) for _ in range(4))
    v = v * v
    plan = T.NewtonSchulzPlan(shapes, DEV)
    a, b = [t.clone() for t in (p, g, m, v)], [t.clone() for t in (p, g, m, v)]

    def both(p, g, m, v):
        T.muon_step(p, g, m, plan, lr=1e-2, weight_decay=0.1)
        T.adamw_step(p, g, m, v, lr=1e-3, step=3)
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both(*[t.clone() for t in a])
    torch.cuda.current_stream().wait_stream(s)
    with torch.cuda.graph(graph):
        both(*a)
    for i in range(4):
        graph.replay()
        both(*b)
        torch.cuda.synchronize()
        for x, y in zip(a, b):
            assert torch.equal(x, y), i
        a[1].mul_(1.5)
        b[1].mul_(1.5)


def test_large_offsets():
    """matrices past 2^31 bytes of a flat buffer"""
    from das_amd import train_ops as T
    far = (1 << 29) + 8 * 12345        # elements: 2 GiB and some
    shapes, offsets = [(1, 100, 70), (1, 80, 300)], [far, far + 7000]
    n = far + 7000 + 24000
    p, g, m = (torch.zeros(n, device=DEV) for _ in range(3))
    gen = torch.Generator().manual_seed(2)
    tail = [torch.randn(31000, generator=gen).to(DEV) for _ in range(3)]
    for t, x in zip((p, g, m), tail):
        t[far:] = x
    T.muon_step(p, g, m, T.NewtonSchulzPlan(shapes, DEV, offsets=offsets), lr=0.1)
    near = [t.clone() for t in tail]
    T.muon_step(*near, T.NewtonSchulzPlan(shapes, DEV), lr=0.1)
    for t, x in zip((p, g, m), near):
        assert torch.equal(t[far:], x) and not t[:far].any()


def test_train_cli_with_muon(tmp_path):
    """tools/train.py with optimizer.type=Muon: trains, checkpoints, resumes"""
    import os
    from test_cli_gpu import run
    work = str(tmp_path / 'w')
    args = ['model.backbone.num_stages=1', 'data.samples_per_gpu=2', 'data.train.type=SyntheticPoseDataset', 'data.train.length=4',
            'data.train.img_shape=(128,192)', 'log_config.interval=1', 'optimizer.type=Muon', 'optimizer.adamw_lr=0.0005',
            'optimizer.momentum=0.95']
    run('tools/train.py', 'configs/das/exp_panoptic.py', '--work-dir', work, '--no-validate', '--cfg-options', *args, 'runner.max_epochs=1')
    ck = os.path.join(work, 'epoch_1.pth')
    sd = torch.load(ck, map_location='cpu', weights_only=False)['optimizer']
    i = sd['das_names'].index('backbone.top.top.0.conv.weight')
    assert sd['das_steps'] == 2 and sd['state'][i]['momentum_buffer'].shape == (64, 3, 7, 7)
    out = run('tools/train.py', 'configs/das/exp_panoptic.py', '--work-dir', work, '--no-validate', '--resume-from', ck, '--cfg-options',
              *args, 'runner.max_epochs=2')
    assert 'Epoch [2]' in out and 'nan' not in out
    sd = torch.load(os.path.join(work, 'epoch_2.pth'), map_location='cpu', weights_only=False)['optimizer']
    assert sd['das_steps'] == 4
