"""CPU: what layer norm, log probabilities and the orthogonalised updates refuse, at the Python entry points and at the C ABI
(nothing is launched: every check comes before the first launch)."""
import ctypes

import pytest
import torch

from luminoth_amd import _lib
from luminoth_amd import kernels as K

Err = _lib.LuminothHipError
F, H, D = torch.float32, torch.float16, torch.float64


def z(*shape, dtype=F):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize('call,text', [
    (lambda: K.layer_norm_fwd(z(4, 8)), 'ROCm device'),
    (lambda: K.layer_norm_fwd(z(4, 8, dtype=D)), 'float32, float16 or bfloat16'),
    (lambda: K.layer_norm_fwd(z(4, 0)), 'at least one column'),
    (lambda: K.layer_norm_fwd(torch.tensor(1.0)), 'at least one column'),
    (lambda: K.layer_norm_fwd(z(8, 4).t()), 'even distance'),
    (lambda: K.layer_norm_fwd(z(8, 4, 6)[:, :3]), 'even distance'),
    (lambda: K.layer_norm_fwd(z(1, 8).expand(4, 8)), 'even distance'),
    (lambda: K.layer_norm_fwd(z(4, 8), z(7)), 'parameters of shape'),
    (lambda: K.layer_norm_fwd(z(4, 8), z(8, dtype=H)), 'parameters in'),
    (lambda: K.layer_norm_fwd(z(4, 8, dtype=H), z(8), z(8, dtype=H)), 'two types'),
    (lambda: K.layer_norm_bwd(z(4, 7), z(4, 8), z(4), z(4)), 'dy like x'),
    (lambda: K.layer_norm_bwd(z(4, 8, dtype=H), z(4, 8), z(4), z(4)), 'dy like x'),
    (lambda: K.layer_norm_bwd(z(4, 8), z(4, 8), z(3), z(4)), 'mean of the forward'),
    (lambda: K.layer_norm_bwd(z(4, 8), z(4, 8), z(4), z(4), addend=z(4, 8), need_dx=False), 'addend needs dx'),
    (lambda: K.layer_norm_bwd(z(4, 8), z(4, 8), z(4), z(4), addend=z(1, 8)), 'addend like x'),
    (lambda: K.log_probs_fwd(z(4, 8)), 'ROCm device'),
    (lambda: K.log_probs_fwd(z(4, 8), top_k=9), 'alternatives'),
    (lambda: K.log_probs_fwd(z(4, 80), top_k=65), 'alternatives'),
    (lambda: K.log_probs_fwd(z(4, 8), top_k=-1), 'alternatives'),
    (lambda: K.log_probs_fwd(z(4, 8), z(4)), 'int32 or int64'),
    (lambda: K.log_probs_fwd(z(4, 8), z(3, dtype=torch.int64)), 'int32 or int64'),
    (lambda: K.log_probs_fwd(z(4, 8, dtype=torch.int32)), 'float32, float16'),
    (lambda: K.log_probs_fwd(z(8, 4).t(), None), 'even distance'),
    (lambda: K.log_probs_bwd(z(4, 8), None, z(4), z(4), g_logp=z(4)), 'targets'),
    (lambda: K.log_probs_bwd(z(4, 8), None, z(4), None, g_entropy=z(4)), 'entropy'),
    (lambda: K.log_probs_bwd(z(4, 8), None, z(3), z(4)), 'lse of shape'),
    (lambda: K.log_probs_bwd(z(4, 8), None, z(4), z(4), top_index=z(4, 2), g_top=z(4, 2)), 'alternatives'),
    (lambda: K.orthogonalize([z(4, 8)]), 'ROCm device'),
    (lambda: K.orthogonalize([z(8)]), 'matrices expected'),
    (lambda: K.orthogonalize([z(8, 0)]), 'matrices expected'),
    (lambda: K.orthogonalize([z(8, 4), z(8, 4, dtype=H)]), 'one type'),
    (lambda: K.orthogonalize([z((1 << 17) + 1, 1)]), 'at most'),
    (lambda: K.orthogonalize([z(4, 8)], steps=0), 'steps'),
    (lambda: K.orthogonalize([z(4, 8)], eps=0.0), 'eps'),
    (lambda: K.muon_step([z(4, 8)], [z(4, 8)], [z(4, 8)], lr=0.1), 'ROCm device'),
    (lambda: K.muon_step([z(4, 8)], [z(4, 8)], [], lr=0.1), 'as many'),
    (lambda: K.muon_step([], [], [], lr=0.1), 'as many'),
    (lambda: K.muon_step([z(4, 8)], [z(8, 4)], [z(4, 8)], lr=0.1), 'one shape'),
    (lambda: K.muon_step([z(4, 8, dtype=H)], [z(4, 8)], [z(4, 8)], lr=0.1), 'float32 expected'),
    (lambda: K.muon_step([z(4, 8)], [z(4, 8)], [z(4, 8)], lr=0.1, factors=z(2)), 'one factor'),
])
def test_refusals(call, text):
    with pytest.raises(Err, match=text):
        call()


def test_muon_refuses_shared_memory():
    w, g, v = z(4, 8), z(4, 8), z(4, 8)
    flat = z(80)
    for params, grads, moms, factors, text in (([w, w], [g, g], [v, z(4, 8)], None, 'weights and momenta overlap'),
                                               ([w], [g], [w], None, 'weights and momenta overlap'),
                                               ([flat[:32].view(4, 8)], [g], [flat[24:56].view(4, 8)], None, 'weights and momenta overlap'),
                                               ([w], [v], [v], None, 'gradients or factors overlap'),
                                               ([w], [w], [v], None, 'gradients or factors overlap'),
                                               ([flat[40:72].view(4, 8)], [flat[16:48].view(4, 8)], [v], None, 'gradients or factors overlap'),
                                               ([w], [g], [v], [v.view(-1)[:1]], 'gradients or factors overlap'),
                                               ([w, z(4, 8)], [g, g], [v, z(4, 8)], [flat[:1], flat[:1]], 'ROCm device')):
        with pytest.raises(Err, match=text):
            K.muon_step(params, grads, moms, lr=0.1, factors=factors)


def test_c_entries_refuse_before_they_launch():
    lib = _lib.load()
    buf = (ctypes.c_float * 64)()
    p = ctypes.cast(buf, ctypes.c_void_p)
    ln = lambda **k: lib.lmh_layer_norm_fwd(k.get('x', p), k.get('ld', 8), None, None, k.get('dt', 0), k.get('pd', 0),      # noqa: E731
                                            k.get('rows', 2), k.get('cols', 8), k.get('eps', 1e-5), p, p, p, None)
    for bad in (dict(x=None), dict(ld=7), dict(dt=3), dict(dt=0, pd=1), dict(dt=1, pd=2), dict(rows=-1), dict(cols=0),
                dict(cols=-4), dict(eps=-1.0), dict(eps=float('nan')), dict(cols=2 ** 30 + 1, ld=2 ** 31)):
        assert ln(**bad) == -1, bad
    assert ln(rows=0) == 0
    bwd = lambda **k: lib.lmh_layer_norm_bwd(p, k.get('lddy', 8), p, 8, k.get('add', None), 8, p, p, None, 0, 0, 2, 8, k.get('dx', p),  # noqa: E731
                                             k.get('dg', p), None, k.get('ws', p), k.get('n', 0), None)
    assert bwd(lddy=3) == -1 and bwd(dx=None, add=p) == -1 and bwd() == -3 and bwd(ws=None, n=4096) == -3
    lp = lambda **k: lib.lmh_log_probs_fwd(k.get('x', p), k.get('ld', 8), k.get('dt', 0), k.get('t', None), 1, k.get('rows', 2),  # noqa: E731
                                           k.get('cols', 8), k.get('top', 0), k.get('lp', None), p, p, k.get('tl', p), k.get('ti', p),
                                           k.get('ws', p), k.get('n', 1 << 20), None)
    for bad in (dict(x=None), dict(ld=7), dict(dt=-1), dict(t=p), dict(lp=p), dict(top=9), dict(cols=100, ld=100, top=65), dict(top=-1),
                dict(top=2, tl=None), dict(top=2, ti=None), dict(rows=-3), dict(rows=2 ** 40), dict(rows=2 ** 24 - 1)):
        assert lp(**bad) == -1, bad
    assert lp(cols=40000, ld=40000, n=0) == -3 and lp(cols=40000, ld=40000, ws=None) == -3 and lp(rows=0) == 0
    lb = lambda **k: lib.lmh_log_probs_bwd(p, 8, 0, k.get('t', None), 1, k.get('lse', p), k.get('h', p), k.get('gl', None),      # noqa: E731
                                           k.get('gh', None), k.get('ti', None), k.get('gt', None), 2, 8, k.get('top', 0), p, None)
    for bad in (dict(lse=None), dict(gl=p), dict(gh=p, h=None), dict(top=2), dict(top=2, ti=p)):
        assert lb(**bad) == -1, bad
    job = (_lib.MuonJob * 1)()
    job[0].rows, job[0].cols = 4, 8
    need = lib.lmh_muon_workspace_bytes(job, 1)
    assert need > 0
    orth = lambda n=1, dt=0, steps=5, eps=1e-7, ws=p, size=need: lib.lmh_orthogonalize(job, n, dt, steps, eps, ws, size, None)   # noqa: E731
    for bad in (dict(n=0), dict(n=-1), dict(dt=3), dict(steps=0), dict(steps=65), dict(eps=0.0), dict(eps=float('nan')), dict()):
        assert orth(**bad) == -1, bad                      # (the last: no input and no output)
    assert orth(ws=None) == -3 and orth(size=need // 2) == -3
    assert lib.lmh_muon_step(job, 1, 5, 1e-7, 1.0, 0.9, 1, 0.1, p, need, None) == -1
    for rows, cols in ((0, 8), (4, -1), ((1 << 17) + 1, 1), (1 << 16, 1 << 15)):
        job[0].rows, job[0].cols = rows, cols
        assert lib.lmh_muon_workspace_bytes(job, 1) == 0 and orth() == -1


def small_store():
    from luminoth_amd.params import ParamStore
    st = ParamStore()
    zeros = lambda shape, gen: torch.zeros(shape)                                  # noqa: E731
    for name, shape, wd in (('a/conv/weights', (3, 3, 4, 8), 0.1), ('a/conv/beta', (8,), 0.0), ('a/conv/gamma', (8,), 0.0),
                            ('b/fc/w', (10, 6), 0.2), ('b/fc/b', (6,), 0.0), ('b/col/w', (9, 1), 0.0), ('b/out/w', (6, 3), 0.0)):
        st.add(name, shape, zeros, wd=wd)
    return st.build('cpu')


def test_muon_takes_the_matrices_and_adam_the_rest():
    from luminoth_amd.utils import training as T
    from luminoth_amd.utils.config import get_config

    class Model(object):
        store = small_store()

    def make(**opt):
        cfg = get_config({'model': {'type': 'fasterrcnn'}, 'train': {'optimizer': dict(opt, _replace=True, type='muon')}})
        return T.get_optimizer(cfg.train, Model)
    opt = make(exclude=['out'])
    assert (opt.momentum, opt.use_nesterov, opt.ns_steps) == (0.95, True, 5)
    assert opt.matrices == ['a/conv/weights', 'b/fc/w']
    off = Model.store.offsets
    assert [(a, b) for a, b, _, _ in opt.adam_runs] == [(1, 3), (4, 7)]
    assert [lo for _, _, lo, _ in opt.adam_runs] == [off['a/conv/beta'][1], off['b/fc/b'][1]]
    for (a, b, lo, hi), (seg, wd) in zip(opt.adam_runs, opt._run_tables):
        assert int(seg[0]) == 0 and int(seg[-1]) == hi - lo and wd.numel() == b - a
    assert opt.adam_runs[-1][3] == Model.store.flat.numel()
    assert make(momentum=0.8, use_nesterov=False, ns_steps=3).ns_steps == 3 and 'b/out/w' in make().matrices
    with pytest.raises(TypeError, match='decay'):
        make(decay=0.9)
    with pytest.raises(ValueError, match='ns_steps'):
        make(ns_steps=0)
    with pytest.raises(Err, match='ROCm device'):
        opt.step()
