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
