"""CPU: what bench.py chooses for launched ranks: from what the machine and the caller export, and from a measured collective."""
import importlib.util
import os
import sys

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

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


def _slow_rank(rank, world, port, q):
    sys.path.insert(0, ROOT)
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    dist.init_process_group('gloo', rank=rank, world_size=world)
    import time
    from luminoth_amd.utils import training
    if rank == 1:                 # this rank's clock says 50 ms more for every interval: a collective with a large fixed cost
        real, calls = time.perf_counter, [0]

        def late():
            calls[0] += 1
            return real() + 0.05 * calls[0]
        time.perf_counter = late
    p = training.allreduce_probe(16 << 20, torch.device('cpu'), reps=2)
    q.put((rank, p['bucket_bytes_from_probe'], p['alpha_us'], [m['ms'] for m in p['messages']]))
    dist.destroy_process_group()


def test_ranks_agree_on_the_bucket_they_measured():
    """Two ranks that measure different times: one bucket size (different ones make collectives of different lengths, which abort or
    hang), that of the slower rank; what each measured itself is still reported."""
    ctx = mp.get_context('spawn')
    q = ctx.Queue()
    procs = [ctx.Process(target=_slow_rank, args=(r, 2, 33500 + os.getpid() % 2000, q)) for r in range(2)]
    for p in procs:
        p.start()
    (_, b0, a0, ms0), (_, b1, a1, ms1) = sorted(q.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    assert b0 == b1 and a0 == a1 and a1 >= 20e3, (b0, b1, a0, a1)
    assert min(ms1) >= 50 and ms0 != ms1


@pytest.mark.parametrize('bucket,gradient,used', [(12, 112, 12), (56, 112, 56), (57, 112, 28), (64, 112, 28), (24, 60, 24), (31, 60, 15), (64, 1000, 64),
                                                  (10, 40, 10), (8, 16, 8), (9, 16, 4), (4, 1, 4), (64, 9, 4)])
def test_a_bucket_leaves_something_to_overlap(bucket, gradient, used):
    """MB: only a bucket of more than half the gradient is cut, to a quarter; what a measured collective asks for below that stays"""
    from luminoth_amd.utils.training import bucket_that_overlaps
    assert bucket_that_overlaps(bucket << 20, gradient << 20) == used << 20
