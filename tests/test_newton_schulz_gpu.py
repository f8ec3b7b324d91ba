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
