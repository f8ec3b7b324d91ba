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
