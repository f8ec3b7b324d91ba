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
