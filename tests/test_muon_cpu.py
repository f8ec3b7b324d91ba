"""Host side of Muon and AdamW: schedules of the Newton-Schulz products, parameter groups, state dicts, config options. No GPU."""
import ctypes as C
import os

import numpy as np
import pytest
import torch
import torch.multiprocessing as mp
import torch.nn as nn

COEF = (3.4445, -4.7750, 2.0315)
MAT = np.dtype([('src', '<i8'), ('x', '<i8'), ('a', '<i8'), ('rows', '<i4'), ('cols', '<i4'), ('m', '<i4'), ('n', '<i4'), ('ldx', '<i4'),
                ('lda', '<i4'), ('group', '<i4'), ('index', '<i4'), ('chunk0', '<i4'), ('chunks', '<i4'), ('scale', '<f4'),
                ('gscale', '<f4'), ('tall', '<i4'), ('thin', '<i4')])
ITEM = np.dtype([(k, '<i4') for k in ('matrix', 'ti', 'tj', 'k0', 'kn', 'slot', 'slots', 'm', 'ldx', 'lda')] +
                [('scale', '<f4'), ('gscale', '<f4'), ('x', '<i8'), ('a', '<i8')])


def make_plan(shapes, steps=5, coef=COEF, offsets=None, eps=1e-7):
    from das_amd import _lib
    lib = _lib.load()
    arr, at = (_lib.DasNsShape * len(shapes))(), 0
    for i, (a, (k, r, c)) in enumerate(zip(arr, shapes)):
        a.off, a.count, a.rows, a.cols = (at if offsets is None else offsets[i]), k, r, c
        at += k * r * c
    plan, cf = _lib.DasNsPlan(), (C.c_float * (3 * steps))(*(list(coef) * steps))
    st = lib.das_ns_plan(arr, len(shapes), steps, cf, eps, C.byref(plan), None, 0)
    if st:
        return st, None, None
    buf = np.zeros(plan.table_bytes, dtype=np.uint8)
    assert lib.das_ns_plan(arr, len(shapes), steps, cf, eps, C.byref(plan), buf.ctypes.data, plan.table_bytes - 1) == _lib.DAS_ERR_ARG
    assert lib.das_ns_plan(arr, len(shapes), steps, cf, eps, C.byref(plan), buf.ctypes.data, plan.table_bytes) == 0
    return 0, plan, buf


def table(buf, at, n, dt):
    return buf[at:at + n * dt.itemsize].view(dt)


@pytest.mark.parametrize('shapes', [[(1, 64, 64)], [(3, 45, 256), (1, 65, 64), (2, 700, 513), (1, 1, 4096), (2, 9000, 33)], [(1, 257, 8192)],
                                    [(2, 2048, 2048), (28, 256, 2304), (6, 512, 4608), (50, 64, 64)], [(5, 1536, 1000)]])
def test_schedule_covers_every_product_once(shapes):
    """every tile of every matrix, every part of its inner axis, exactly once; offsets inside the work areas"""
    st, plan, buf = make_plan(shapes)
    assert st == 0 and MAT.itemsize == 80
    mats = table(buf, plan.mat_at, plan.n_matrices, MAT)
    end = plan.n_matrices - plan.n_thin
    assert (mats['m'][:plan.n_small] <= 64).all() and not mats['thin'][:end].any()
    assert (mats['m'][plan.n_small:end] > 64).all() and (mats['m'][end:] <= 64).all() and mats['thin'][end:].all()
    assert plan.n_matrices == sum(s[0] for s in shapes) and plan.small_lds <= 155 * 1024
    assert sorted(zip(mats['rows'], mats['cols'])) == sorted((r, c) for k, r, c in shapes for _ in range(k))
    for part, x_elems, a_elems in ((mats[plan.n_small:end], plan.x_elems, plan.a_elems), (mats[end:], plan.thin_x_elems, plan.thin_a_elems)):
        for lead, area, size in (('x', 'ldx', x_elems), ('a', 'lda', a_elems)):
            spans = sorted((int(o), int(o) + int(m) * int(ld)) for o, m, ld in zip(part[lead], part['m'], part[area]))
            assert all(e <= s for (_, e), (s, _) in zip(spans, spans[1:])) and (not spans or spans[-1][1] <= size)
    slices = table(buf, plan.slice_at, plan.n_slices, ITEM)
    for q, (first, count) in enumerate(table(buf, plan.thin_at, 2 * plan.n_thin, np.dtype('<i4')).reshape(-1, 2)):
        M, mine = mats[end + q], slices[first:first + count]
        frags = (-(-M['m'] // 16)) ** 2
        assert (mine['matrix'] == end + q).all() and count <= 64 and mine['k0'][0] == 0
        assert (mine['k0'][1:] == mine['k0'][:-1] + mine['kn'][:-1]).all() and (mine['k0'][-1] + mine['kn'][-1]) * 128 == M['ldx']
        assert (mine['slot'] == mine['slot'][0] + frags * np.arange(count)).all() and mine['slot'][-1] + frags <= plan.thin_slots
    assert sum(table(buf, plan.thin_at, 2 * plan.n_thin, np.dtype('<i4')).reshape(-1, 2)[:, 1]) == plan.n_slices
    chunks = table(buf, plan.chunk_at, plan.n_chunks, np.dtype([(k, '<i4') for k in 'qrci']))
    assert len(set(map(tuple, chunks[['q', 'r', 'c']].tolist()))) == plan.n_chunks
    for at, n, join_at, n_join, slots, tile, inner in (
            (plan.gram_at, plan.n_gram, plan.gram_join_at, plan.n_gram_join, plan.gram_slots, plan.gram_tile, 'ldx'),
            (plan.product_at, plan.n_product, plan.product_join_at, plan.n_product_join, plan.product_slots, plan.product_tile, 'lda')):
        seen, used = {}, []
        for t in table(buf, at, n, ITEM):
            if t['matrix'] < 0:
                continue
            assert t['kn'] > 0 and t['ti'] >= t['tj']
            assert all(t[k] == mats[t['matrix']][k] for k in ('m', 'ldx', 'lda', 'scale', 'gscale', 'x', 'a'))
            seen.setdefault((t['matrix'], t['ti'], t['tj']), []).append((t['k0'], t['kn'], t['slot']))
        joins = {(t['matrix'], t['ti'], t['tj']): t for t in table(buf, join_at, n_join, ITEM)}
        want = {(q, i, j) for q in range(plan.n_small, end) for i in range(-(-mats[q]['m'] // tile)) for j in range(i + 1)}
        assert set(seen) == want
        for key, parts in seen.items():
            parts.sort()
            assert parts[0][0] == 0 and sum(p[1] for p in parts) * 64 == mats[key[0]][inner]
            assert all(a[0] + a[1] == b[0] for a, b in zip(parts, parts[1:]))
            if key in joins:
                first, count = joins[key]['slot'], joins[key]['slots']
                assert [p[2] for p in parts] == list(range(first, first + count))
                used += [p[2] for p in parts]
            else:
                assert len(parts) == 1 and parts[0][2] == -1
        assert len(set(used)) == len(used) and (not used or max(used) < slots)
    seen = [(t['matrix'], t['ti'], t['tj']) for t in table(buf, plan.update_at, plan.n_update, ITEM) if t['matrix'] >= 0]
    T = plan.update_tile
    want = {(q, i, j) for q in range(plan.n_small, end) for i in range(-(-mats[q]['m'] // T)) for j in range(mats[q]['ldx'] // T)}
    assert len(seen) == len(set(seen)) and set(seen) == want


def test_plan_refusals():
    ok = [(1, 8, 8)]
    assert make_plan(ok)[0] == 0
    for bad in (lambda: make_plan([(0, 8, 8)]), lambda: make_plan([(1, 0, 8)]), lambda: make_plan([(1, 8, -1)]),
                lambda: make_plan([(1, 8, (1 << 20) + 1)]), lambda: make_plan([(1, 40000, 40000)]), lambda: make_plan(ok, eps=-1.0),
                lambda: make_plan(ok, eps=float('nan')), lambda: make_plan(ok, steps=17), lambda: make_plan(ok, coef=(float('inf'), 0, 0)),
                lambda: make_plan(ok, coef=(50.0, 0.0, 0.0)), lambda: make_plan(ok, steps=8, coef=(2.0, 0.0, 0.0)),
                lambda: make_plan([(1, 8, 8), (1, 8, 8)], offsets=[0, 60]), lambda: make_plan(ok, offsets=[-8])):
        assert bad()[0] == 1
    assert make_plan([(1, 8, 8), (1, 8, 8)], offsets=[64, 0])[0] == 0


def test_plan_limits():
    """what a launch's grid, the offsets' arithmetic and the polynomial's forms bear"""
    assert make_plan([(1 << 22, 2, 2)])[0] == 1 and make_plan([(1 << 20, 2, 2)])[0] == 0
    assert make_plan([(1, 8, 8)], offsets=[(1 << 60) + 1])[0] == 1
    assert make_plan([(1, 8, 8)], offsets=[(1 << 63) - 8])[0] == 1
    st, plan, _ = make_plan([(1, 8, 8)], offsets=[1 << 60])
    assert st == 0 and plan.extent == (1 << 60) + 64


def test_overlapping_buffers_are_refused():
    """by the library, before any launch: a step would read elements that it has already written"""
    from das_amd import _lib
    lib = _lib.load()
    _, plan, _ = make_plan([(1, 8, 8)])
    base, far = 1 << 20, 1 << 24
    for p, g, b in ((base, base, far), (base, far, base + 4), (far, base + 252, base), (base + 16, far, base)):
        assert lib.das_muon_step(C.byref(plan), 4096, p, g, b, 1e-2, 0.9, 0.0, 1, 0, 1.0, 0.0, None, 8192, None) == _lib.DAS_ERR_ARG
    for bufs in ((base, base, far, 2 * far), (base, far, 2 * far, base + 252), (base, far, far + 4, 2 * far), (base, base + 256, far, far + 128)):
        assert lib.das_adamw_step(*bufs, 64, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, 0.0, None, None) == _lib.DAS_ERR_ARG


def test_phases_follow_the_polynomial():
    """steps on the Gram matrix end before an error of it can have grown 256-fold: three, then two of the default polynomial; a cubic
    whose slope at zero is 1.5 may go further"""
    _, plan, _ = make_plan([(1, 300, 300)])
    assert list(plan.phase_end)[:5] == [3, 4, 5, 5, 5]
    _, plan, _ = make_plan([(1, 300, 300)], steps=12, coef=(1.5, -0.5, 0.0))
    assert plan.phase_end[0] == 7 and plan.phase_end[11] == 12


def test_ops_refuse_cpu_tensors():
    from das_amd import train_ops as T
    from das_amd._lib import DasHipError
    t = torch.zeros(8, 8)
    for bad in (lambda: T.orthogonalize(t), lambda: T.orthogonalize([t]), lambda: T.adamw_step(t, t, t, t, lr=1e-3, step=1),
                lambda: T.muon_step(t, t, t, None, lr=1e-3), lambda: T.NewtonSchulzPlan([(8, 8)], 'cpu')):
        with pytest.raises(DasHipError):
            bad()


def net():
    torch.manual_seed(0)
    return nn.Sequential(nn.Conv2d(3, 16, 3), nn.BatchNorm2d(16), nn.Conv2d(16, 45, 1), nn.Conv2d(48, 2, 1), nn.Linear(64, 24), nn.Linear(3, 64))


def test_muon_parameter_groups():
    from das_amd.optim import build_optimizer
    m = net()
    want = {k: v.clone() for k, v in m.state_dict().items()}
    opt = build_optimizer(m, dict(optimizer=dict(type='Muon', lr=0.02, weight_decay=0.1, adamw_lr=1e-3, adamw_weight_decay=0.01,
                                                 adamw_params=['0.weight'], paramwise_cfg=dict(bias_lr_mult=2., bias_decay_mult=0.)),
                                  optimizer_config=dict(grad_clip=dict(max_norm=35))))
    group_of = {n: next(g['key'] for g in opt.groups if g['start'] <= sl.off < g['end']) for n, sl in zip(opt._names, opt.slots)}
    assert group_of == {'0.weight': 'main', '0.bias': 'bias', '1.weight': 'main', '1.bias': 'main', '2.weight': 'matrix', '2.bias': 'bias',
                        '3.weight': 'main', '3.bias': 'bias', '4.weight': 'matrix', '4.bias': 'bias', '5.weight': 'main', '5.bias': 'bias'}
    for k, v in m.state_dict().items():
        assert torch.equal(v, want[k])
    by = {g['key']: g for g in opt.groups}
    assert by['matrix']['start'] == opt.flat_v.numel() and by['matrix']['end'] == opt.flat_p.numel()
    lrs = {g['key']: (round(o['lr'], 6), o['weight_decay']) for g, o in zip(opt.groups, opt.param_groups)}
    assert lrs == {'matrix': (0.02, 0.1), 'main': (0.001, 0.01), 'bias': (0.002, 0.0)} and opt.max_grad_norm == 35
    assert opt.buckets[-1][1] == opt.flat_p.numel()


@pytest.mark.parametrize('kind', ['AdamW', 'Muon'])
def test_state_dict_round_trip(kind):
    from das_amd.optim import build_optimizer
    cfg = dict(type=kind, lr=1e-3, weight_decay=0.1)
    a, b = build_optimizer(net(), cfg), build_optimizer(net(), cfg)
    assert a.state_dict()['state'] == {}
    for o in (a,):
        for n, sl in zip(o._names, o.slots):
            o.flat_m[sl.off:sl.off + sl.numel].normal_()
            if sl.off < o.flat_v.numel():
                o.flat_v[sl.off:sl.off + sl.numel].uniform_()
        o.steps = 7
    sd = a.state_dict()
    assert len(sd['param_groups']) == len(list(net().parameters())) and all(g['params'] == [i] for i, g in enumerate(sd['param_groups']))
    b.load_state_dict(sd)
    assert torch.equal(a.flat_m, b.flat_m) and torch.equal(a.flat_v, b.flat_v) and b.steps == 7
    i = sd['das_names'].index('2.weight')
    key = 'exp_avg' if kind == 'AdamW' else 'momentum_buffer'
    assert sd['state'][i][key].shape == (45, 16, 1, 1) and sd['state'][i][key].is_contiguous()
    other = build_optimizer(net(), dict(type='Muon' if kind == 'AdamW' else 'AdamW', lr=1e-3))
    with pytest.raises(ValueError):
        other.load_state_dict(sd)
    with pytest.raises(ValueError):
        b.load_state_dict(dict(sd, param_groups=sd['param_groups'][1:]))


def test_adamw_state_dict_is_torchs():
    from das_amd.optim import FlatAdamW
    m = net()
    topt = torch.optim.AdamW(m.parameters(), lr=1e-3, betas=(0.9, 0.95), weight_decay=0.1)
    for p in m.parameters():
        p.grad = torch.randn_like(p)
    topt.step()
    topt.step()
    opt = FlatAdamW(net(), lr=1e-3, betas=(0.9, 0.95), weight_decay=0.1)
    opt.load_state_dict(topt.state_dict())
    assert opt.steps == 2
    dense = opt._dense_momentum()
    for n, p in m.named_parameters():
        assert torch.equal(dense[n], topt.state[p]['exp_avg'])
    m2 = net()
    back = torch.optim.AdamW([dict(params=[p]) for p in m2.parameters()], lr=1.0)
    sd = opt.state_dict()
    back.load_state_dict(dict(state=sd['state'], param_groups=sd['param_groups']))
    for p, q in zip(m.parameters(), m2.parameters()):
        for k in ('exp_avg', 'exp_avg_sq'):
            assert torch.equal(topt.state[p][k], back.state[q][k])
        assert float(back.state[q]['step']) == 2 and back.param_groups[0]['lr'] == 1e-3 and back.param_groups[0]['betas'] == (0.9, 0.95)


def test_config_refusals():
    from das_amd.optim import FlatAdamW, FlatMuon, build_optimizer
    for cfg in (dict(type='AdamW', lr=1e-3, momentum=0.9), dict(type='Muon', lr=1e-3, beta=0.9), dict(type='AdamW'),
                dict(type='Muon', lr=1e-3, lr_scale='rms'), dict(type='Muon', lr=0.0), dict(type='Muon', lr=1e-3, momentum=1.0),
                dict(type='AdamW', lr=1e-3, betas=(0.9, 1.0)), dict(type='AdamW', lr=1e-3, eps=0.0),
                dict(type='AdamW', lr=1e-3, paramwise_cfg=dict(norm_decay_mult=0.))):
        with pytest.raises(ValueError):
            build_optimizer(net(), cfg)
    with pytest.raises(AssertionError):
        build_optimizer(net(), dict(type='Adam', lr=1e-3))
    from das_amd._lib import DasHipError
    for cls in (FlatAdamW, FlatMuon):       # no CPU fallback
        with pytest.raises(DasHipError):
            cls(net(), lr=1e-3).step()


def _worker(rank, port, ret):
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port))
    dist.init_process_group('gloo', rank=rank, world_size=2)
    from das_amd.optim import FlatMuon
    m = net()
    opt = FlatMuon(m, lr=0.1, bucket_mb=0)
    ok = opt.world == 2 and len(opt.buckets) > 1
    for i, p in enumerate(m.parameters()):
        p.grad.fill_(float(rank + 1) * (i + 1))
    opt.all_reduce_grads()
    ok &= all(torch.equal(p.grad, torch.full_like(p.grad, 3.0 * (i + 1))) for i, p in enumerate(m.parameters()))
    ret[rank] = ok
    dist.destroy_process_group()


def test_muon_gradients_are_summed_over_two_ranks():
    mp.set_start_method('spawn', force=True)
    ret = mp.Manager().dict()
    mp.spawn(_worker, args=(30500 + os.getpid() % 1000, ret), nprocs=2, join=True)
    assert ret[0] and ret[1]
