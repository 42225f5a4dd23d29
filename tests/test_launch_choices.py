"""CPU: what bench.py chooses for a launched rank from what the machine and the caller export."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def bench():
    spec = importlib.util.spec_from_file_location('bench_choices', os.path.join(ROOT, 'bench.py'))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize('exported,used', [(None, '8'), ('', '8'), ('4', '8'), ('8', '8'), ('2', '2'), ('1', '1'), ('6', '6'), ('16', '16'),
                                           ('default', 'default')])
def test_hardware_queues(exported, used):
    """Unset, or HIP's default that a machine exports for everybody: eight; a caller's own number, and what is no number, stays."""
    assert bench().hardware_queues(exported) == used
