"""Host side of the Newton-Schulz plans and of the optimizers built on them: what is refused, where host memory lies. No GPU."""
import pytest
import torch


class Recorder:
    """the library, with the calls of das_ns_plan noted"""

    def __init__(self):
        from das_amd import _lib
        self.lib, self.tables = _lib.load(), []

    def __getattr__(self, name):
        return getattr(self.lib, name)

    def das_ns_plan(self, *a):
        self.tables.append(a[6].value if a[6] is not None else None)
        return self.lib.das_ns_plan(*a)


@pytest.mark.parametrize('shapes', [[(8, 8)], [(20000, 2, 3)]])     # (the second: tables larger than the first guess)
def test_plan_tables_are_host_memory_whatever_the_default_device(monkeypatch, shapes):
    """das_ns_plan writes the tables from the host: a tensor of the default device would be GPU memory that kernels still use"""
    from das_amd import _lib
    from das_amd import train_ops as T
    rec = Recorder()
    monkeypatch.setattr(_lib, 'load', lambda: rec)
    with torch.device('meta'):      # (tensors of this device have no memory: their address is null)
        try:
            T.NewtonSchulzPlan(shapes, 'cuda:0')
        except (RuntimeError, AssertionError):
            pass                    # (no GPU to copy the tables to)
    assert rec.tables and rec.tables[0] and rec.tables[-1]


def test_arguments_beside_a_plan_have_to_agree_with_it():
    """(on a plan without tables: no GPU)"""
    from das_amd import train_ops as T
    from das_amd._lib import DasHipError
    plan = T.NewtonSchulzPlan([(0, 5)], 'cuda:0', steps=4, eps=1e-6)
    for kw in (dict(steps=5), dict(eps=1e-7), dict(coefficients=(1.5, -0.5, 0.0)), dict(coefficients=[T.NS_COEFFICIENTS] * 5)):
        with pytest.raises(DasHipError):
            plan._agrees(**{**dict(steps=None, coefficients=None, eps=None), **kw})
    plan._agrees(None, None, None)
    plan._agrees(4, [T.NS_COEFFICIENTS] * 4, 1e-6)


def nets():
    """with matrices and the rest, and with matrices alone"""
    import torch.nn as nn
    torch.manual_seed(0)
    yield lambda: nn.Sequential(nn.Conv2d(8, 16, 3), nn.BatchNorm2d(16), nn.Linear(64, 24))
    yield lambda: nn.Sequential(nn.Linear(64, 24, bias=False), nn.Linear(24, 64, bias=False))


def filled(opt, steps):
    with torch.no_grad():
        for sl in opt.slots:
            opt.flat_m[sl.off:sl.off + sl.numel].normal_()
            if hasattr(opt, 'flat_v') and sl.off < opt.flat_v.numel():
                opt.flat_v[sl.off:sl.off + sl.numel].uniform_()
    opt.steps = steps
    return opt


@pytest.mark.parametrize('which', [0, 1])
@pytest.mark.parametrize('src', ['SGD', 'AdamW', 'Muon'])
@pytest.mark.parametrize('dst', ['SGD', 'AdamW', 'Muon'])
def test_state_of_another_optimizer_is_refused_whole(src, dst, which):
    """no moment of one kind becomes a momentum of another, and a refused file leaves every buffer as it was"""
    from das_amd.optim import build_optimizer
    net = list(nets())[which]
    sd = filled(build_optimizer(net(), dict(type=src, lr=1e-2)), 3).state_dict()
    opt = filled(build_optimizer(net(), dict(type=dst, lr=1e-2)), 5)
    before = [opt.flat_m.clone()] + ([opt.flat_v.clone()] if hasattr(opt, 'flat_v') else [])
    if src == dst:
        opt.load_state_dict(sd)
        assert opt.steps == 3 and not torch.equal(opt.flat_m, before[0])
        return
    with pytest.raises(ValueError):
        opt.load_state_dict(sd)
    assert opt.steps == 5 and torch.equal(opt.flat_m, before[0]) and (len(before) == 1 or torch.equal(opt.flat_v, before[1]))


def test_state_that_does_not_fit_is_refused_whole():
    from das_amd.optim import build_optimizer
    for kind in ('AdamW', 'Muon'):
        net = list(nets())[0]
        sd = filled(build_optimizer(net(), dict(type=kind, lr=1e-2)), 3).state_dict()
        opt = filled(build_optimizer(net(), dict(type=kind, lr=1e-2)), 5)
        m, v = opt.flat_m.clone(), opt.flat_v.clone()
        last = len(sd['param_groups']) - 1
        for bad in ({k: t[..., :-1] if k != 'step' else t for k, t in sd['state'][last].items()}, {'step': torch.tensor(3.0)}):
            with pytest.raises(ValueError):
                opt.load_state_dict(dict(sd, state={**sd['state'], last: bad}))
            assert torch.equal(opt.flat_m, m) and torch.equal(opt.flat_v, v) and opt.steps == 5


def test_state_of_torchs_optimizers():
    """torch.optim.SGD's state goes into SGD, torch.optim.AdamW's into AdamW, each with one group for all parameters; a file without state anywhere"""
    from das_amd.optim import build_optimizer
    for net in nets():
        for make, kind in ((lambda p: torch.optim.SGD(p, lr=0.1, momentum=0.9), 'SGD'), (lambda p: torch.optim.AdamW(p, lr=0.1), 'AdamW')):
            m = net()
            topt = make(m.parameters())
            fresh = topt.state_dict()
            for p in m.parameters():
                p.grad = torch.randn_like(p)
            topt.step()
            for other in ('SGD', 'AdamW', 'Muon'):
                opt = build_optimizer(net(), dict(type=other, lr=1e-2))
                opt.load_state_dict(fresh)
                assert opt.steps == 0 and not opt.flat_m.any()
                if other == kind:
                    opt.load_state_dict(topt.state_dict())
                    dense = opt._dense_momentum()
                    for n, p in m.named_parameters():
                        assert torch.equal(dense[n], topt.state[p]['momentum_buffer' if kind == 'SGD' else 'exp_avg'])
                else:
                    with pytest.raises(ValueError):
                        opt.load_state_dict(topt.state_dict())


def test_sizes_past_the_librarys_integers_are_refused():
    """a count of 2^32 + 1 is not one matrix, and a set too large for a launch is a refusal, not a want of host memory"""
    from das_amd import train_ops as T
    from das_amd._lib import DasHipError
    for shapes, kw in (([((1 << 32) + 1, 1, 1)], {}), ([(1, (1 << 32) + 8, 8)], {}), ([(8, (1 << 32) + 8)], {}), ([(8, 8)], dict(offsets=[1 << 64])),
                       ([(8, 8)], dict(offsets=[(1 << 64) + 64])), ([(1 << 21, 1 << 14, 1 << 14)], {})):
        with pytest.raises(DasHipError):
            T.NewtonSchulzPlan(shapes, 'cuda:0', **kw)


@pytest.mark.parametrize('names', ['2.w', ['2.w'], ('2.w', 'nothing')])
def test_adamw_params_is_one_name_or_several(names):
    """(a name alone is not its letters: '2.w' is part of no other name, but '.' is part of all)"""
    from das_amd.optim import build_optimizer
    opt = build_optimizer(list(nets())[0](), dict(type='Muon', lr=1e-2, adamw_params=names))
    by = {n: next(g['key'] for g in opt.groups if g['start'] <= sl.off < g['end']) for n, sl in zip(opt._names, opt.slots)}
    assert by['0.weight'] == 'matrix' and by['2.weight'] == 'main'


@pytest.mark.parametrize('rank', [1, 16, 0])
@pytest.mark.parametrize('shape', [(1, 64), (64, 64), (30, 3000), (300, 200)])
def test_the_bounds_reject_wrong_results(monkeypatch, shape, rank):
    """the limits of the GPU tests of five steps, on the CPU: zeros, the negated result, the normalised input, a step too few or too many and a tile
    of 16 x 16 left out are all far outside; the result in f32 and its bf16 rounding are inside"""
    import test_newton_schulz_gpu as g
    monkeypatch.setattr(g, 'DEV', 'cpu')
    u = g.low_rank(*shape, rank, 3)
    ref = g.polar64(u)
    limit, half = g.pairs_bound(min(shape), rank or min(shape)), (g.pairs_bound(min(shape), rank or min(shape)) ** 2 + 2.0 ** -16 / 3) ** 0.5
    hole = ref.clone()
    i = int(ref.abs().argmax())
    hole[i // shape[1] // 16 * 16:][:16, i % shape[1] // 16 * 16:][:, :16] = 0
    for wrong in (torch.zeros_like(ref), -ref, u.double() / u.double().norm(), g.polar64(u, steps=4), g.polar64(u, steps=6), hole):
        assert g.off(wrong, u) > 5 * half > 5 * limit
    assert g.off(ref.float(), u) <= limit and g.off(ref.bfloat16(), u) <= half
