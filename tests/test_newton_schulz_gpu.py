"""Newton-Schulz orthogonalisation and the Muon step: values at measured accuracy, plans' lifetimes, rarely used ways to call them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
COEF = (3.4445, -4.7750, 2.0315)


def test_default_device_of_the_gpu_changes_nothing():
    """(a plan's tables are made in host memory, also where torch makes tensors on the GPU by itself)"""
    from das_amd import train_ops as T
    u = torch.randn(3, 80, 200, generator=torch.Generator().manual_seed(0)).to(DEV)
    want = T.orthogonalize(u)
    with torch.device('cuda'):
        got = T.orthogonalize(u)
    assert torch.equal(got, want)


@pytest.mark.parametrize('muon', [False, True])
def test_plan_dropped_while_another_stream_reads_its_tables(muon):
    """the tables' memory is handed out again only when the calls that read it have ended"""
    from das_amd import train_ops as T
    u = torch.randn(200, 300, generator=torch.Generator().manual_seed(0)).to(DEV)
    p, m, want = torch.zeros(60000, device=DEV), torch.zeros(60000, device=DEV), torch.zeros(60000, device=DEV)
    plan = T.NewtonSchulzPlan([(200, 300)], DEV)
    if muon:
        T.muon_step(want, u.view(-1), m, plan, lr=0.1)
        m.zero_()
    else:
        want = T.orthogonalize([u], plan=plan)[0]
    tables = plan._flat[1]
    at, size = tables.data_ptr(), tables.numel()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(1 << 24)          # (the call below is still waiting when the plan goes)
        if muon:
            T.muon_step(p, u.view(-1), m, plan, lr=0.1)
            got = p
        else:
            got = T.orthogonalize([u], plan=plan)[0]
    del plan, tables
    fresh = [torch.full((size,), 255, dtype=torch.uint8, device=DEV) for _ in range(16)]
    early = any(f.data_ptr() <= at < f.data_ptr() + size for f in fresh) and not s.query()
    s.synchronize()
    assert not early and torch.equal(got, want)


@pytest.mark.parametrize('shape', [(600, 700), (900, 500), (1, 64, 5000), (3000, 48), (16, 64, 256), (40, 30, 64)])
def test_every_element_keeps_its_22_bits(shape):
    """One step of the polynomial x -> x: an element leaves as it went in, but for its two roundings to a pair of f16 (2^-22 each of it, and the
    2^-25 of f16's subnormal numbers over the scale, at least sqrt(n / 2)), the f32 factor, its product, the sum that it is alone in and the norm
    (f32 sums of squares of 24 additions, under a root): 2^-19 = (2 * 4 + 24) 2^-24 covers them. A wrong low part is 2^-11."""
    from das_amd import train_ops as T
    u = torch.randn(shape, generator=torch.Generator().manual_seed(shape[-1])).to(DEV)
    u = u * torch.exp(torch.randn(shape[:-1], generator=torch.Generator().manual_seed(5)))[..., None].to(DEV)
    got = T.orthogonalize(u, steps=1, coefficients=(1.0, 0.0, 0.0), out_dtype=torch.float32).double()
    x = u.double() / (torch.linalg.matrix_norm(u.double())[..., None, None] + 1e-7)
    off = (got - x).abs()
    assert (off <= 2.0 ** -19 * x.abs() + 2.0 ** -25 / (max(shape[-2:]) / 2) ** 0.5).all(), float((off / x.abs()).max())


@pytest.mark.parametrize('shape', [(64, 200), (40, 7000), (1500, 1500), (600, 5000)])
def test_small_elements_keep_their_bits_too(shape):
    """As above, of a rank-one matrix, whose elements are about (m n)^-1/2. The polynomial x -> x keeps X's norm at one, so that X is stored times
    2^15 and a subnormal number is 2^-25 2^-15 off; the first pass stores blocks with their largest element at 2^9 or more: 2^-34 of it."""
    from das_amd import train_ops as T
    gen = torch.Generator().manual_seed(shape[1])
    u = torch.outer(torch.randn(shape[0], generator=gen), torch.randn(shape[1], generator=gen)).to(DEV)
    got = T.orthogonalize(u, steps=1, coefficients=(1.0, 0.0, 0.0), out_dtype=torch.float32).double()
    x = u.double() / (u.double().norm() + 1e-7)
    off = (got - x).abs()
    assert (off <= 2.0 ** -19 * x.abs() + 2.0 ** -40 + 2.0 ** -34 * x.abs().max()).all(), float((off / x.abs()).max())


def low_rank(r, c, k, seed):
    """a weight's gradient out of k pixels: channels of very different size times rectified features; for k = 0 out of more than the sides"""
    gen = torch.Generator().manual_seed(seed)
    k = k or 2 * max(r, c)
    d = torch.randn(k, r, generator=gen) * torch.exp(torch.randn(r, generator=gen))
    x = (torch.randn(k, c, generator=gen) + torch.randn(k, 1, generator=gen)).relu()
    return d.to(DEV).t() @ x.to(DEV)


def polar64(u, coef=COEF, steps=5, eps=1e-7):
    """the formula in 64 bits"""
    x = u.double() / (u.double().norm() + eps)
    x = x.t() if x.shape[0] > x.shape[1] else x
    a, b, c = coef
    for _ in range(steps):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if u.shape[0] > u.shape[1] else x


def off(got, u, **kw):
    """distance from the formula over its norm (2-norm over all entries)"""
    ref = polar64(u, **kw)
    return float((got.double() - ref).norm() / ref.norm())


def pairs_bound(m, rank):
    """Error of an f32 result of five default steps over the result's norm. What X is off outside its row and column space grows by 3.4445 a
    step: 485 in all; the result's `rank` singular values are 0.7 at least. X is rounded to a pair three times on its way (as it comes in, divided
    by its norm, after the first phase), by at most 2^-23 of an element each time, uniform in that: 3^-1/2 of it on the average of a matrix,
    2^-23 for the three. Each of the two products Q X adds 3 m / 32 partial sums of m inner elements one after the other, in f32, half a step
    (2^-24) at most each, again uniform: 2^-24 (m / 32)^1/2 a product. Errors of Q and G stay in X's row space and do not grow."""
    return 3.4445 ** 5 / 0.7 * (2.0 ** -46 + 2 * m / 32 * 2.0 ** -48) ** 0.5 / min(rank or 16, 16) ** 0.5


@pytest.mark.parametrize('rank', [1, 2, 16, 0])
@pytest.mark.parametrize('shape', [(64, 64), (60, 64), (30, 3000), (3000, 20), (256, 2304), (700, 513), (1024, 1024), (4096, 4096), (2048, 8192)],
                         ids=lambda s: '%dx%d' % s)
def test_f32_result_of_any_rank(shape, rank):
    from das_amd import train_ops as T
    u = low_rank(*shape, rank, seed=sum(shape) + rank)
    assert off(T.orthogonalize(u, out_dtype=torch.float32), u) <= pairs_bound(min(shape), rank)


@pytest.mark.parametrize('out_dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('rank', [1, 4, 16, 128, 0])
@pytest.mark.parametrize('shape', [(60, 64), (30, 3000), (256, 2304), (1030, 900), (2048, 2048)], ids=lambda s: '%dx%d' % s)
def test_16_bit_result_is_the_f32_one_rounded(shape, rank, dtype, out_dtype):
    """... so that it is off by its rounding alone: half a step, uniform in that, 3^-1/2 of it on the average; f16's subnormal numbers are half of
    2^-24 apart, whatever the element"""
    from das_amd import train_ops as T
    u = low_rank(*shape, rank, seed=sum(shape) + rank)
    u = (u / u.abs().max()).to(dtype)
    got, f32 = T.orthogonalize(u, out_dtype=out_dtype), T.orthogonalize(u, out_dtype=torch.float32)
    ref = polar64(u)
    half = torch.finfo(out_dtype).eps / 2
    tiny = 2.0 ** -25 * (shape[0] * shape[1] / 3) ** 0.5 / float(ref.norm()) if out_dtype == torch.float16 else 0
    # (a 16-bit input is of full rank, by its own rounding, and counted as the f32 matrix that it came from)
    assert off(got, u) <= (pairs_bound(min(shape), rank) ** 2 + half ** 2 / 3 + tiny ** 2) ** 0.5
    assert torch.equal(got, f32.to(out_dtype))


def test_arguments_beside_a_plan():
    """a plan has its steps, polynomial and eps: other ones are refused, the same ones are not"""
    from das_amd import train_ops as T
    from das_amd._lib import DasHipError
    u = torch.randn(70, 90, generator=torch.Generator().manual_seed(0)).to(DEV)
    plan = T.NewtonSchulzPlan([(70, 90)], DEV)
    want = T.orthogonalize([u], plan=plan)[0]
    for kw in (dict(steps=3), dict(coefficients=(1.5, -0.5, 0.0)), dict(coefficients=[COEF] * 4), dict(eps=1e-3), dict(steps=5, eps=0.0)):
        with pytest.raises(DasHipError):
            T.orthogonalize([u], plan=plan, **kw)
    for kw in (dict(steps=5), dict(coefficients=COEF), dict(coefficients=[COEF] * 5, eps=1e-7), dict(steps=None)):
        assert torch.equal(T.orthogonalize([u], plan=plan, **kw)[0], want)
    assert torch.equal(T.orthogonalize([u])[0], want) and torch.equal(T.orthogonalize([u], steps=5, coefficients=COEF, eps=1e-7)[0], want)


@pytest.mark.parametrize('shape', [(30, 50), (30, 4000), (200, 100)])
@pytest.mark.parametrize('momentum', [0.98, 0.95, 0.9])
def test_muons_average_is_as_exact_as_f32(momentum, shape):
    """mu m + (1 - mu) g: the two factors, the two products and the sum are rounded once each, half a step (2^-24) at most, of terms whose sum of sizes
    is |mu m| + |(1 - mu) g|: three of them on either way"""
    from das_amd import train_ops as T
    gen = torch.Generator().manual_seed(1)
    n = shape[0] * shape[1]
    p, g, m = (torch.randn(n, generator=gen).to(DEV) for _ in range(3))
    m[::2] = 0
    a, b = momentum * m.double(), (1 - momentum) * g.double()
    T.muon_step(p, g, m, T.NewtonSchulzPlan([shape], DEV), lr=0.1, momentum=momentum)
    assert ((m.double() - (a + b)).abs() <= 3 * 2.0 ** -24 * (a.abs() + b.abs())).all()


# sets whose launches are of every form: (tile side, wave groups a tile, whether inner axes are split) of X X^T and of the m x m products, (tile side,
# wave groups) of Q X; odd and ragged sizes
FORMS = [([(1, 256, 2304)], (64, 4, True), (64, 4, False), (64, 4)),
         ([(8, 145, 1547)], (64, 4, True), (64, 4, False), (128, 2)),
         ([(12, 141, 1616), (9, 227, 1084)], (64, 4, False), (64, 4, False), (128, 1)),
         ([(2, 998, 981)], (128, 2, True), (64, 4, False), (64, 4)),
         ([(5, 530, 370), (6, 729, 387)], (128, 2, True), (64, 4, False), (128, 2)),
         ([(9, 597, 929), (3, 284, 1781)], (128, 2, True), (128, 2, False), (128, 1)),
         ([(2, 1805, 867), (12, 1164, 386)], (128, 2, True), (128, 2, True), (128, 1)),
         ([(1, 2048, 2048)], (128, 2, False), (128, 2, False), (128, 2)),
         ([(12, 297, 1921), (10, 974, 929)], (128, 1, True), (128, 1, False), (128, 1)),
         ([(5, 802, 1142), (1, 1981, 186), (11, 918, 1057), (3, 64, 64), (2, 30, 3000), (1, 5000, 12)], (128, 1, True), (128, 1, True), (128, 1)),
         ([(5, 64, 64), (2, 1, 256), (3, 30, 3000), (1, 5000, 12), (2, 64, 257)], None, None, None)]


def stacks(shapes, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    out = []
    for k, r, c in shapes:
        pix = 2 * max(r, c)
        d = torch.randn(k, r, pix, generator=gen, device=DEV) * torch.exp(torch.randn(k, r, 1, generator=gen, device=DEV))
        x = (torch.randn(k, pix, c, generator=gen, device=DEV) + torch.randn(k, pix, 1, generator=gen, device=DEV)).relu()
        out.append(d @ x)
    return out


def polar64_stack(u, steps, coef=COEF):
    x = u.double() / (torch.linalg.matrix_norm(u.double())[:, None, None] + 1e-7)
    x = x.mT.contiguous() if x.shape[1] > x.shape[2] else x
    a, b, c = coef
    for _ in range(steps):
        g = x @ x.mT.contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.mT if u.shape[1] > u.shape[2] else x


def check_stack(got, u, ref, what):
    """every matrix of a stack; fewer steps than five lose less than pairs_bound has"""
    d = torch.linalg.matrix_norm(got.double() - ref) / torch.linalg.matrix_norm(ref)
    limit = pairs_bound(min(u.shape[1:]), min(u.shape[1:]))
    assert (d <= limit).all(), (what, tuple(u.shape), d.tolist(), limit)


@pytest.mark.parametrize('steps', [1, 2, 3, 4, 5])
@pytest.mark.parametrize('form', range(len(FORMS)))
def test_every_form_of_the_launches(form, steps):
    """every matrix of sets that reach every kernel, with the forms named so that another schedule shows; Muon's results by a parameter of zero that
    becomes -f X; bf16 results"""
    from das_amd import train_ops as T
    shapes, gram, product, update = FORMS[form]
    plan = T.NewtonSchulzPlan(shapes, DEV, steps=steps)
    p = plan._flat[0]
    if gram:
        assert (p.gram_tile, p.gram_kg, p.n_gram_join > 0) == gram and (p.update_tile, p.update_kg) == update
        assert (p.product_tile, p.product_kg, p.n_product_join > 0) == product
    mats = stacks(shapes, form)
    refs = [polar64_stack(u, steps) for u in mats]
    got = T.orthogonalize(mats, plan=plan, out_dtype=torch.float32)
    for u, y, ref in zip(mats, got, refs):
        check_stack(y, u, ref, 'f32')
    for y, z in zip(got, T.orthogonalize(mats, plan=plan)):
        assert torch.equal(z, y.bfloat16())
    g = torch.cat([u.reshape(-1) for u in mats])
    w, m = torch.zeros_like(g), torch.zeros_like(g)
    T.muon_step(w, g, m, plan, lr=1.0, momentum=0.0, nesterov=False)
    assert torch.equal(m, g)
    at = 0
    for u, ref in zip(mats, refs):
        f = max(1.0, u.shape[1] / u.shape[2]) ** 0.5
        check_stack(-w[at:at + u.numel()].view(u.shape) / f, u, ref, 'muon')
        at += u.numel()


@pytest.mark.parametrize('shape', [(60, 64), (50, 1200), (96, 160), (300, 200)], ids=lambda s: '%dx%d' % s)
@pytest.mark.parametrize('kind', ['1e-30', '1e-12', '1e12', '1e30', 'spike', 'decay', 'strides', 'transposed', 'expanded', 'bf16 view'])
def test_five_steps_on_hard_inputs(kind, shape):
    """magnitudes at f32's ends, one entry over all, singular values over twelve decades, strides and starts: by the bound of a rank-one result"""
    from das_amd import train_ops as T
    r, c = shape
    u, eps = low_rank(r, c, 0, 7), 1e-7
    if kind[0] == '1':
        u, eps = u / u.norm() * float(kind), 0.0 if float(kind) < 1 else 1e-7
    elif kind == 'spike':
        u = 1e-6 * u / u.norm()
        u[r - 1, c - 1] = 1e6
    elif kind == 'decay':
        a, _, b = torch.linalg.svd(u.cpu().double(), full_matrices=False)
        u = (a * torch.logspace(0, -12, min(r, c), dtype=torch.float64) @ b).float().to(DEV)
    elif kind == 'strides':
        u = low_rank(2 * r + 1, c + 7, 0, 7)[1::2, 3:-4]
    elif kind == 'transposed':
        u = low_rank(c, r, 0, 7).t()
    elif kind == 'expanded':
        u = u[:1].expand(r, -1)
    elif kind == 'bf16 view':
        u = low_rank(r, c + 1, 0, 7).bfloat16()[:, 1:]
    assert u.shape == shape
    got = T.orthogonalize(u, eps=eps, out_dtype=torch.float32)
    assert off(got, u, eps=eps) <= pairs_bound(min(shape), 1)
    assert torch.equal(T.orthogonalize(u, eps=eps), got.bfloat16())


def x_bound(x, m):
    """2-norm error of X out of a Muon step: pairs_bound's for what grows (times 0.7, the norm it is over there), the same relative to X for what does
    not; U's own rounding, four halves of an f32 step, grows like X's"""
    return 0.7 * pairs_bound(m, 1) + pairs_bound(m, 16) * float(x.norm()) + 3.4445 ** 5 * 4 * 2.0 ** -24


@pytest.mark.parametrize('nesterov,lr_scale', [(True, 'original'), (False, 'match_rms_adamw'), (True, 'match_rms_adamw')])
@pytest.mark.parametrize('rank', [1, 16, 0])
def test_muon_step_with_momentum_and_decay(nesterov, lr_scale, rank):
    from das_amd import train_ops as T
    shapes = [(64, 147), (300, 70), (1, 256), (30, 3000), (700, 513)]
    n = sum(r * c for r, c in shapes)
    gen = torch.Generator().manual_seed(rank)
    g = torch.cat([low_rank(r, c, rank, 1).reshape(-1) for r, c in shapes])
    m = 0.5 * torch.cat([low_rank(r, c, rank, 2).reshape(-1) for r, c in shapes])
    p = torch.randn(n, generator=gen).to(DEV)
    mu, lr, wd = 0.95, 0.5, 0.1
    m64 = mu * m.double() + (1 - mu) * g.double()
    u64 = (1 - mu) * g.double() + mu * m64 if nesterov else m64
    p64 = p.double() * (1 - lr * wd)
    T.muon_step(p, g, m, T.NewtonSchulzPlan(shapes, DEV), lr=lr, momentum=mu, weight_decay=wd, nesterov=nesterov, lr_scale=lr_scale)
    at = 0
    for r, c in shapes:
        s = slice(at, at + r * c)
        at += r * c
        x = polar64(u64[s].view(r, c))
        f = max(1.0, r / c) ** 0.5 if lr_scale == 'original' else 0.2 * max(r, c) ** 0.5
        d = float((p[s].double() - p64[s] + lr * f * x.reshape(-1)).norm())
        assert d <= lr * f * x_bound(x, min(r, c)) + 4 * 2.0 ** -24 * float(p64[s].norm() + lr * f * x.norm()), (r, c)


def test_flat_muon_moves_a_detectors_matrices_by_their_orthogonal_factors():
    """two clipped steps of a small detector: what each matrix moved by, over the learning rate, against 64 bits"""
    from das_amd.optim import build_optimizer
    from test_train_step_gpu import make
    model, data = make('f32')
    opt = build_optimizer(model, dict(optimizer=dict(type='Muon', lr=0.01, weight_decay=0.1, momentum=0.9, adamw_lr=1e-3),
                                      optimizer_config=dict(grad_clip=dict(max_norm=35))))
    group = next(g for g in opt.groups if g['key'] == 'matrix')
    mats = [(n, p, sl) for n, p, sl in zip(opt._names, opt._params, opt.slots) if group['start'] <= sl.off < group['end']]
    assert len(mats) > 20
    m64 = {n: torch.zeros(sl.numel, dtype=torch.float64, device=DEV) for n, _, sl in mats}
    moved = 0
    for _ in range(2):
        opt.zero_grad()
        model.train_step(data, None)['loss'].backward()
        opt.all_reduce_grads()
        before, g = opt.flat_p.double(), opt.flat_g.double()
        k = min(1.0, 35 / (float(g.norm()) + 1e-6))
        opt.step(0.01)
        for n, p, sl in mats:
            s, r, c = slice(sl.off, sl.off + sl.numel), p.shape[0], p.numel() // p.shape[0]
            m64[n] = 0.9 * m64[n] + 0.1 * k * g[s]
            x = polar64((0.1 * k * g[s] + 0.9 * m64[n]).view(r, c))
            f = max(1.0, r / c) ** 0.5
            got = (before[s] * (1 - 0.01 * 0.1) - opt.flat_p[s].double()) / (0.01 * f)
            # (the clip factor's own error scales U, which its norm takes out but for eps)
            limit = x_bound(x, min(r, c)) + 2.0 ** -16 * float(x.norm()) + 3 * 2.0 ** -24 * float(before[s].norm()) / (0.01 * f)
            assert float((got - x.reshape(-1)).norm()) <= limit, n
            moved += float(x.norm()) > 0.5
    assert moved > 30


def test_second_stream_beside_small_tiles():
    """a chain of small and thin matrices beside 64 x 64 tiles: the same bits as captured, where one stream does all, with sources and results reused
    at once behind the call"""
    from das_amd import train_ops as T
    shapes = [(1, 700, 513), (3, 64, 64), (2, 27, 2304), (1, 64, 5000)]
    mats = stacks(shapes, 1)
    plan = T.NewtonSchulzPlan(shapes, DEV)
    assert plan._flat[0].product_tile == 64 and plan._flat[0].n_product >= 32 and plan._flat[0].n_small and plan._flat[0].n_thin
    static, graph = [t.clone() for t in mats], torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        want = T.orthogonalize(static, plan=plan, out_dtype=torch.float32)
    graph.replay()
    for _ in range(20):
        buf = [t.clone() for t in mats]
        got = T.orthogonalize(buf, plan=plan, out_dtype=torch.float32)
        for b in buf:
            b.zero_()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    for u, y in zip(mats, got):
        check_stack(y, u, polar64_stack(u, 5), 'second stream')
