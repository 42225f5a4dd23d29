"""Layer norm, log probabilities and orthogonalised updates as they are used together: the RCNN head with `layer_norm`, its
`top_alternatives`, the `muon` optimizer of a model, and a classifier trained with all three against float64."""
import math

import numpy as np
import pytest
import torch

from luminoth_amd import autograd as A
from luminoth_amd import kernels as K

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)


def orthogonal(u):
    x = u / max(float(torch.linalg.norm(u)), 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    for _ in range(5):
        g = x @ x.t()
        x = COEF[0] * x + (COEF[1] * g + COEF[2] * (g @ g)) @ x
    return x.t() if tall else x


def make_model(optimizer=None, clip=False, **rcnn):
    from e2e_util import condition_like_pretrained
    from luminoth_amd.models import get_model
    from luminoth_amd.utils.config import get_config
    cfg = get_config({'model': {'type': 'fasterrcnn', 'network': {'num_classes': 20},
                                'base_network': {'architecture': 'resnet_v1_50'}, 'rcnn': rcnn},
                      'train': {'seed': 0, 'clip_by_norm': clip, 'optimizer': dict(optimizer or {'type': 'momentum', 'momentum': 0.9}, _replace=True),
                                'learning_rate': {'_replace': True, 'decay_method': None, 'learning_rate': 1e-3}}})
    return cfg, condition_like_pretrained(get_model('fasterrcnn')(cfg), 'resnet_v1_50')


def norm_ref(x, gamma, beta):
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    return (x - mean) / (var + 1e-5).sqrt() * gamma + beta


def test_head_with_layer_norm(monkeypatch):
    """The gradients of every variable of the head, from the fused train step, against autograd in float64 of the same stack from
    the same pooled features and loss gradients; the module API's path gives the same."""
    from e2e_util import synth
    cfg, model = make_model(layer_sizes=[192, 100], layer_norm=True)
    r = model._rcnn
    names = [v for l in r.layers for v in (l.w_name, l.b_name)] + [v for n in r._norms for v in n]
    assert names[-1] == 'fasterrcnn/rcnn/fc_1/LayerNorm/beta' and all(n in model.store.grads for n in names)
    g = torch.Generator().manual_seed(0)
    for n in r._norms:                                     # values that matter
        model.store[n[0]].copy_(1 + 0.3 * torch.randn(model.store[n[0]].shape, generator=g))
        model.store[n[1]].copy_(0.3 * torch.randn(model.store[n[1]].shape, generator=g))
    seen = {}
    plain = r.train_bwd

    def spy(ctx, d_cls, d_off, *a, **k):
        seen.update(net=ctx['steps'][0][2].clone(), d_cls=d_cls.clone(), d_off=d_off.clone(), cls=ctx['cls_score'].clone())
        return plain(ctx, d_cls, d_off, *a, **k)
    monkeypatch.setattr(r, 'train_bwd', spy)
    images, gts = synth(2, 256, 320, 3, 20, 13)
    model.train_step(images, gts)
    torch.cuda.synchronize()
    got = {n: model.store.grads[n].clone() for n in names}

    p = {n: model.store[n].detach().cpu().double().requires_grad_() for n in names}
    x = seen['net'].cpu().double()
    for l, n in zip(r._layers, r._norms):
        x = norm_ref((x @ p[l.w_name] + p[l.b_name]).clamp(0, 6), p[n[0]], p[n[1]])
    cls = x @ p[r._classifier_layer.w_name] + p[r._classifier_layer.b_name]
    off = x @ p[r._bbox_layer.w_name] + p[r._bbox_layer.b_name]
    # products over up to 1024 features and 512 rows in float32: 2^-24 sqrt(1024) of a result, a few of them in a row
    tol = 16 * 32 * 2.0 ** -24
    close = lambda a, b: float(torch.linalg.norm(a.cpu().double().reshape(b.shape) - b)) <= tol * float(torch.linalg.norm(b)) + 1e-12   # noqa: E731
    assert close(seen['cls'], cls.detach())
    ((cls * seen['d_cls'].cpu().double().reshape(cls.shape)).sum() + (off * seen['d_off'].cpu().double().reshape(off.shape)).sum()).backward()
    for n in names:
        assert close(got[n], p[n].grad), n

    monkeypatch.setattr(r, 'train_bwd', plain)
    cfg, other = make_model(layer_sizes=[192, 100], layer_norm=True)
    other.load_state_dict(model.state_dict())
    pred = other(images, gts, is_training=True)
    other.backward(other.loss(pred))
    for n in names:
        assert close(other.store.grads[n], got[n].cpu().double()), n


def test_alternatives_of_the_head():
    from e2e_util import synth
    cfg, model = make_model(layer_sizes=[64], layer_norm=True, top_alternatives=3)
    images, _ = synth(2, 256, 320, 3, 20, 13)
    pred = model(images, is_training=False)['classification_prediction']
    alt, score = pred['rcnn']['alternatives'], pred['rcnn']['cls_score'].detach().cpu().double()
    lp = torch.log_softmax(score, -1)
    assert alt['classes'].shape == score.shape[:2] + (3,) and alt['entropy'].shape == score.shape[:2]
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :3]
    assert torch.equal(alt['classes'].cpu(), order)
    assert float((alt['log_probs'].cpu().double() - lp.gather(-1, order)).abs().max()) <= 200 * 2.0 ** -24
    assert float((alt['entropy'].cpu().double() + (lp.exp() * lp).sum(-1)).abs().max()) <= 1000 * 2.0 ** -24
    assert (alt['classes'][..., 0] == pred['rcnn']['cls_prob'].argmax(-1)).float().mean() > 0.99     # (ties apart)
    with pytest.raises(ValueError, match='top_alternatives'):
        make_model(top_alternatives=22)


@pytest.mark.parametrize('clip', [False, True])
def test_muon_updates_a_model(clip):
    """One optimizer step of the whole detector: every matrix by the formula in float64, everything else by Adam's."""
    from e2e_util import synth
    from luminoth_amd.utils import training as T
    cfg, model = make_model({'type': 'muon', 'exclude': ['fc_bbox']}, clip=clip, layer_sizes=[96], layer_norm=True)
    opt = T.get_optimizer(cfg.train, model)
    assert isinstance(opt, T.MuonOptimizer)
    st = model.store
    rest = [n for n in st.trainable_names() if n not in opt.matrices]
    assert 'fasterrcnn/rcnn/fc_bbox/w' in rest and 'fasterrcnn/rcnn/fc_0/LayerNorm/gamma' in rest and 'fasterrcnn/rpn/conv/w' in opt.matrices
    assert all(len(st.specs[n].shape) == 1 or n == 'fasterrcnn/rcnn/fc_bbox/w' for n in rest)
    images, gts = synth(2, 256, 320, 3, 20, 13)
    g = torch.Generator().manual_seed(1)
    st.mom.copy_(torch.randn(st.mom.shape, generator=g) * 1e-3)
    opt._slot2.copy_(torch.rand(st.mom.shape, generator=g) * 1e-4)
    model.train_step(images, gts)
    torch.cuda.synchronize()
    w0, g0, m0, s0 = (t.cpu().double().clone() for t in (st.flat, st.grad, st.mom, opt._slot2))
    opt.global_step = 3
    opt.step()
    torch.cuda.synchronize()
    lr = 1e-3
    for n in st.trainable_names():
        _, o, cnt = st.offsets[n]
        shape = st.specs[n].shape
        at = slice(o, o + cnt)
        gp = g0[at] + st.specs[n].wd * w0[at]
        if clip:
            gp = gp * (10.0 / max(float(torch.linalg.norm(gp)), 10.0))
        if n in opt.matrices:
            v = 0.95 * m0[at] + gp
            u = (gp + 0.95 * v).view(-1, shape[-1])
            step = lr * 0.2 * math.sqrt(max(u.shape)) * orthogonal(u).reshape(-1)
            # the products' bound of 2910 * 2^-22 (1 + sqrt(k) / 64) on O and some roundings of u on top: relative to |O| >= 0.6 sqrt(rank)
            tol = lr * 0.2 * math.sqrt(max(u.shape)) * 2 * 2910 * 2.0 ** -22 * (1 + math.sqrt(max(u.shape)) / 64)
        else:
            v = 0.9 * m0[at] + 0.1 * gp
            s = 0.95 * s0[at] + 0.05 * gp * gp
            step = lr * math.sqrt(1 - 0.95 ** 4) / (1 - 0.9 ** 4) * v / (s.sqrt() + 1e-8)
            tol = 2.0 ** -20 * float(torch.linalg.norm(step))
        err = float(torch.linalg.norm(st.flat[at].cpu().double() - (w0[at] - step)))
        assert err <= tol + 2.0 ** -23 * float(torch.linalg.norm(w0[at])), (n, err, tol)
        assert float(torch.linalg.norm(st.mom[at].cpu().double() - v)) <= 2.0 ** -20 * (float(torch.linalg.norm(v)) + float(torch.linalg.norm(gp))), n


def test_everything_together_trains_through_the_launch_plan():
    """Layer norm in the head, Muon as the optimizer: eager, recorded and replayed steps give what eager steps give."""
    from e2e_util import synth
    from luminoth_amd import plan as P
    from luminoth_amd.utils import training as T
    images, gts = synth(2, 256, 320, 3, 20, 13)
    losses = {}
    for planned in (False, True):
        cfg, model = make_model({'type': 'muon'}, layer_sizes=[96], layer_norm=True, top_alternatives=2)
        opt = T.get_optimizer(cfg.train, model)
        was, P.ENABLED = P.ENABLED, planned
        try:
            losses[planned] = [float(T.train_step(model, opt, images, gts)[0]) for _ in range(6)]
        finally:
            P.ENABLED = was
        plans = [pl for S in model._step_state.values() for pl in S['plans'].values()] if planned else []
        assert not planned or sum(pl.replays for pl in plans) >= 1
        out = model(images, is_training=False)['classification_prediction']['rcnn']['alternatives']
        assert torch.isfinite(out['log_probs']).all() and torch.isfinite(out['entropy']).all()
    assert np.isfinite(losses[True]).all() and losses[True] == losses[False]


def test_a_classifier_with_all_three():
    """Three steps of a two-layer classifier: matrix product, layer norm, matrix product, log probabilities of the labels plus
    entropy and alternatives in the loss, Muon - against the same in float64."""
    g = torch.Generator().manual_seed(0)
    x, t = torch.randn((60, 48), generator=g), torch.randint(0, 37, (60,), generator=g)
    t[::9] = -1
    w1, w2 = torch.randn((48, 80), generator=g) * 0.2, torch.randn((80, 37), generator=g) * 0.2
    gamma, beta = torch.ones(80), torch.zeros(80)
    dev = [v.clone().cuda().requires_grad_() for v in (w1, w2, gamma, beta)]
    ref = [v.clone().double().requires_grad_() for v in (w1, w2, gamma, beta)]
    mom = [torch.zeros_like(v) for v in dev[:2]]
    rmom = [torch.zeros_like(v) for v in ref[:2]]
    for _ in range(3):
        logits = A.layer_norm(x.cuda() @ dev[0], dev[2], dev[3]) @ dev[1]
        logp, entropy, top, index = A.log_probs(logits, t.cuda(), 2)
        (0.1 * top.sum() - logp.sum() - 0.05 * entropy.sum()).backward()
        z = norm_ref(x.double() @ ref[0], ref[2], ref[3]) @ ref[1]
        lp = torch.log_softmax(z, -1)
        best = torch.sort(z, dim=-1, descending=True, stable=True)
        assert torch.equal(best.indices[:, :2], index.cpu())
        want = torch.where(t < 0, 0.0, lp.gather(1, t.clamp(min=0)[:, None])[:, 0])
        (0.1 * lp.gather(1, best.indices[:, :2]).sum() - want.sum() + 0.05 * (lp.exp() * lp).sum()).backward()
        for a, b in zip(dev, ref):
            # float32 products over 80 and 60 terms, a few in a row
            assert float(torch.linalg.norm(a.grad.cpu().double() - b.grad)) <= 2e-5 * float(torch.linalg.norm(b.grad)) + 1e-7
        with torch.no_grad():
            K.muon_step([v.data for v in dev[:2]], [v.grad for v in dev[:2]], mom, lr=0.02)
            for w, v in zip(ref[:2], rmom):
                v.mul_(0.95).add_(w.grad)
                w -= 0.02 * 0.2 * math.sqrt(max(w.shape)) * orthogonal(w.grad + 0.95 * v)
            for a, b in zip(dev[2:], ref[2:]):
                a -= 0.01 * a.grad
                b -= 0.01 * b.grad
            for v in dev + ref:
                v.grad = None
    for a, b in zip(dev, ref):
        # each step moves a weight by lr 0.2 sqrt(80) O: O is off by 2e-5 of its gradient's norm, 485 times over where O is small
        assert float(torch.linalg.norm(a.detach().cpu().double() - b.detach())) <= 3 * 0.02 * 0.2 * 9 * 485 * 2e-5 + 1e-5


def test_calls_from_two_threads():
    """Two threads with a stream each, the same operators at the same time: the bits of the calls alone."""
    import threading
    g = torch.Generator().manual_seed(11)
    inputs = [(torch.randn((300, 1500), generator=g).cuda(), torch.randn((6, 50000), generator=g).bfloat16().cuda(),
               torch.randint(0, 50000, (6,), generator=g).cuda(), [torch.randn((200, 310), generator=g).cuda() for _ in range(2)]) for _ in range(2)]

    def calls(x, logits, targets, mats):
        y, mean, rstd = K.layer_norm_fwd(x)
        dg, db = torch.empty(1500, device='cuda'), torch.empty(1500, device='cuda')
        out = [y, K.layer_norm_bwd(x, x, mean, rstd, None, dg, db), dg, db]
        out += list(K.log_probs_fwd(logits, targets, 5))
        out.append(K.log_probs_bwd(logits, targets, out[-1], out[-4], torch.ones(6, device='cuda')))
        return out + K.orthogonalize(mats)
    want = [calls(*a) for a in inputs]
    torch.cuda.synchronize()
    got, failed = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i].append(calls(*inputs[i]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                              # (pytest sees only its own thread)
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for i in range(2):
        for results in got[i]:
            for a, b in zip(want[i], results):
                assert torch.equal(a, b)
