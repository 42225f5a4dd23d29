"""The operators of a trained head and its optimizer, as plain torch forms and as calls of luminoth_amd.

Layer norm (forward, backward), log probabilities of given classes or tokens with entropy and top alternatives (forward,
forward + backward), and orthogonalised updates (Newton-Schulz products, alone and as a whole optimizer step).  `own`
chooses the side; inputs come from `prepare` alone and are the same for both.
"""
import math

import torch

own = False

TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
SIZE = {'f32': 4, 'f16': 2, 'bf16': 2}
COEF = (3.4445, -4.7750, 2.0315)     # the published quintic
LN_EPS, NS_EPS, NS_STEPS = 1e-5, 1e-7, 5

# The trainable matrices of Faster R-CNN on ResNet-50 with 80 classes (fine_tune_from block2, 12 anchors), in x out, HWIO
# kernels flattened: block2, block3, RPN, RCNN heads.
RESNET50 = ('256x128;256x512;512x128*3;1152x128*4;128x512*4;512x256;512x1024;1024x256*5;2304x256*6;256x1024*6;'
            '9216x512;512x24;512x48;1024x81;1024x320')


def listed():
    return [
        # the RCNN head's rows: 2 images x 256 ROIs of 1024 features, in the framework's own type
        {'name': 'ln_fwd_head_f32', 'op': 'ln_fwd', 'rows': 512, 'cols': 1024, 'pad': 0, 'type': 'f32'},
        # a long batch of wide rows in 16 bits
        {'name': 'ln_fwd_wide_bf16', 'op': 'ln_fwd', 'rows': 16384, 'cols': 4096, 'pad': 0, 'type': 'bf16'},
        # odd columns, rows of a wider buffer
        {'name': 'ln_bwd_odd_f16', 'op': 'ln_bwd', 'rows': 5003, 'cols': 1001, 'pad': 7, 'type': 'f16', 'addend': False},
        # backward of the long batch, the residual branch's gradient added
        {'name': 'ln_bwd_wide_bf16', 'op': 'ln_bwd', 'rows': 16384, 'cols': 4096, 'pad': 0, 'type': 'bf16', 'addend': True},
        # one answer of a large vocabulary, with its alternatives: latency
        {'name': 'lp_one_row_bf16', 'op': 'lp_fwd', 'rows': 1, 'cols': 131072, 'pad': 0, 'type': 'bf16', 'top': 20, 'masked': 0.0},
        # 2 images x 2000 proposals over 80 classes and background
        {'name': 'lp_classes_f32', 'op': 'lp_fwd', 'rows': 4000, 'cols': 81, 'pad': 0, 'type': 'f32', 'top': 5, 'masked': 0.0},
        # a scoring batch over an odd vocabulary inside padded rows, some rows masked
        {'name': 'lp_score_f16', 'op': 'lp_fwd', 'rows': 2048, 'cols': 100003, 'pad': 61, 'type': 'f16', 'top': 8, 'masked': 0.2},
        # training on log probabilities and entropy: forward and the gradient of the logits
        {'name': 'lp_train_bf16', 'op': 'lp_train', 'rows': 4096, 'cols': 65536, 'pad': 0, 'type': 'bf16', 'top': 0, 'masked': 0.0},
        {'name': 'lp_train_odd_f32', 'op': 'lp_train', 'rows': 777, 'cols': 32003, 'pad': 5, 'type': 'f32', 'top': 3, 'masked': 0.1},
        # one small update matrix
        {'name': 'orth_small_bf16', 'op': 'orth', 'matrices': '1024x320', 'type': 'bf16'},
        # a large fully connected layer
        {'name': 'orth_large_f32', 'op': 'orth', 'matrices': '4096x4096', 'type': 'f32'},
        # the whole optimizer step of the default detector
        {'name': 'muon_resnet50', 'op': 'muon', 'matrices': RESNET50, 'type': 'f32', 'nesterov': True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['ln_fwd', 'ln_bwd', 'lp_fwd', 'lp_train', 'orth', 'muon'])
    kind = rng.choice(['f32', 'f16', 'bf16'])
    pad = rng.choice([0, 0, rng.randint(1, 64)])
    if op in ('ln_fwd', 'ln_bwd'):
        cols = _log(rng, 32, 16384)
        if rng.random() < 0.5:
            cols = cols // 8 * 8
        rows = _log(rng, 1, min(65536, 60000000 // cols))
        case = {'op': op, 'rows': rows, 'cols': cols, 'pad': pad, 'type': kind}
        if op == 'ln_bwd':
            case['addend'] = rng.random() < 0.5
        return case
    if op in ('lp_fwd', 'lp_train'):
        cols = _log(rng, 21, 200000)
        if rng.random() < 0.5:
            cols = max(24, cols // 8 * 8)
        rows = _log(rng, 1, min(8192, 150000000 // cols))
        return {'op': op, 'rows': rows, 'cols': cols, 'pad': pad, 'type': kind, 'top': rng.randint(0, 20),
                'masked': rng.choice([0.0, 0.1, 0.5])}
    if op == 'orth':
        m = _log(rng, 16, 2048)
        n = min(16384, int(m * math.exp(rng.uniform(0, math.log(16)))))
        count = rng.randint(1, 4)
        shape = '%dx%d' % ((m, n) if rng.random() < 0.5 else (n, m))
        return {'op': op, 'matrices': shape if count == 1 else '%s*%d' % (shape, count), 'type': kind}
    groups = []
    for _ in range(rng.randint(2, 12)):
        m = _log(rng, 4, 768)
        n = min(9216, int(m * math.exp(rng.uniform(0, math.log(18)))))
        a, b = (m, n) if rng.random() < 0.3 else (n, m)
        groups.append('%dx%d*%d' % (a, b, rng.randint(1, 4)))
    return {'op': op, 'matrices': ';'.join(groups), 'type': 'f32', 'nesterov': rng.random() < 0.7}


def _shapes(text):
    """'1024x256*5;9216x512' -> [(1024, 256, 5), (9216, 512, 1)]"""
    got = []
    for part in text.split(';'):
        size, _, count = part.partition('*')
        rows, cols = (int(v) for v in size.split('x'))
        got.append((rows, cols, int(count or 1)))
    return got


def _padded(rows, cols, pad, gen, kind, scale=1.0):
    """(rows, cols) values; with `pad`, the first columns of wider rows"""
    full = torch.randn((rows, cols + pad), generator=gen, device='cuda') * scale
    return full.to(TYPES[kind])[:, :cols]


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    op, kind = case['op'], case['type']
    s = {'op': op, 'case': case}
    if op in ('ln_fwd', 'ln_bwd'):
        rows, cols = case['rows'], case['cols']
        # features with an offset of their own per row
        x = _padded(rows, cols, case['pad'], gen, 'f32') + torch.randn((rows, 1), generator=gen, device='cuda')
        s['x'] = _like_padded(x, case, kind)
        s['gamma'] = 1 + 0.2 * torch.randn(cols, generator=gen, device='cuda')
        s['beta'] = 0.1 * torch.randn(cols, generator=gen, device='cuda')
        if op == 'ln_bwd':
            s['dy'] = _padded(rows, cols, 0, gen, kind)
            s['addend'] = _padded(rows, cols, 0, gen, kind) if case['addend'] else None
            mean, rstd = _moments(s['x'])
            s['mean'], s['rstd'] = mean, rstd
            s['dgamma'], s['dbeta'] = torch.empty_like(s['gamma']), torch.empty_like(s['beta'])
    elif op in ('lp_fwd', 'lp_train'):
        rows, cols = case['rows'], case['cols']
        x = _padded(rows, cols, case['pad'], gen, kind, 3.0)
        at = torch.randint(0, cols, (rows,), generator=gen, device='cuda')
        if rows > 3:
            at[1::7] = -1                                    # rows whose answer is not asked for
        x[torch.arange(rows, device='cuda'), at.clamp(min=0)] += 4.0          # the model knows something
        if case['masked']:
            # rows where only some classes are allowed (the answer among them), and one where none is
            r = torch.rand((rows, 1), generator=gen, device='cuda') < case['masked']
            drop = torch.rand((rows, cols), generator=gen, device='cuda') < 0.9
            drop[torch.arange(rows, device='cuda'), at.clamp(min=0)] = False
            x.masked_fill_(r & drop, -math.inf)
            if rows > 1:
                x[rows // 2] = -math.inf
        s['x'], s['targets'] = x, at
        if op == 'lp_train':
            s['g_logp'] = torch.randn(rows, generator=gen, device='cuda')
            s['g_entropy'] = 0.1 * torch.randn(rows, generator=gen, device='cuda')
            s['g_top'] = torch.randn((rows, _top(case)), generator=gen, device='cuda') if case['top'] else None
    else:
        # gradients: a few strong directions over noise
        mats = []
        for rows, cols, count in _shapes(case['matrices']):
            r = min(8, rows, cols)
            for _ in range(count):
                strong = torch.randn((rows, r), generator=gen, device='cuda') @ torch.randn((r, cols), generator=gen, device='cuda')
                mats.append(1e-3 * (0.3 * strong + torch.randn((rows, cols), generator=gen, device='cuda')))
        if op == 'orth':
            s['mats'] = [m.to(TYPES[kind]) for m in mats]
        else:
            # one flat buffer each for weights, gradients and momentum, as the parameter store keeps them
            total = sum(m.numel() for m in mats)
            flat = torch.cat([m.reshape(-1) for m in mats])
            s['flat_w'] = 0.05 * torch.randn(total, generator=gen, device='cuda')
            s['flat_v'] = 5e-3 * torch.randn(total, generator=gen, device='cuda') + 3 * flat
            s['flat_g'] = flat
            for key in ('w', 'v', 'g'):
                views, at = [], 0
                for m in mats:
                    views.append(s['flat_' + key][at:at + m.numel()].view(m.shape))
                    at += m.numel()
                s[key] = views
    return s


def _like_padded(x, case, kind):
    full = torch.zeros((case['rows'], case['cols'] + case['pad']), device='cuda', dtype=TYPES[kind])
    full[:, :case['cols']] = x
    return full[:, :case['cols']]


def _moments(x):
    x = x.double()
    mean = x.mean(-1)
    return mean.float(), (1 / ((x - mean[:, None]).square().mean(-1) + LN_EPS).sqrt()).float()


def _top(case):
    return min(case['top'], case['cols'])


MU, LR, WD = 0.95, 0.02, 5e-4


def _scale(rows, cols):
    return 0.2 * math.sqrt(max(rows, cols))


def run(state):
    op = state['op']
    if own:
        return _run_own(state, op)
    if op == 'ln_fwd':
        return _ln_fwd(state['x'].float(), state['gamma'], state['beta'], state['x'].dtype)
    if op == 'ln_bwd':
        return _ln_bwd(state)
    if op == 'lp_fwd':
        return _lp_fwd(state)
    if op == 'lp_train':
        return _lp_train(state)
    if op == 'orth':
        return [o.to(u.dtype) for o, u in zip(_orthogonal([u.float() for u in state['mats']]), state['mats'])]
    return _muon(state)


# ---------------------------------------------------------------- the framework's calls ----
def _run_own(state, op):
    from luminoth_amd import kernels as K
    if op == 'ln_fwd':
        y, mean, rstd = K.layer_norm_fwd(state['x'], state['gamma'], state['beta'], LN_EPS)
        return {'y': y, 'mean': mean, 'rstd': rstd}
    if op == 'ln_bwd':
        dx = K.layer_norm_bwd(state['dy'], state['x'], state['mean'], state['rstd'], state['gamma'], state['dgamma'],
                              state['dbeta'], addend=state['addend'])
        return {'dx': dx, 'dgamma': state['dgamma'], 'dbeta': state['dbeta']}
    if op == 'lp_fwd':
        logp, entropy, top, index, lse = K.log_probs_fwd(state['x'], state['targets'], _top(state['case']))
        return {'logp': logp, 'entropy': entropy, 'lse': lse, 'top': top, 'index': index}
    if op == 'lp_train':
        logp, entropy, top, index, lse = K.log_probs_fwd(state['x'], state['targets'], _top(state['case']))
        dx = K.log_probs_bwd(state['x'], state['targets'], lse, entropy, state['g_logp'], state['g_entropy'], index,
                             state['g_top'])
        return {'logp': logp, 'entropy': entropy, 'top': top, 'index': index, 'dx': dx}
    if op == 'orth':
        return K.orthogonalize(state['mats'], steps=NS_STEPS, eps=NS_EPS)
    K.muon_step(state['w'], state['g'], state['v'], lr=LR, momentum=MU, nesterov=state['case']['nesterov'],
                weight_decay=WD, steps=NS_STEPS, eps=NS_EPS)
    return {'w': state['flat_w'], 'v': state['flat_v']}


# -------------------------------------------------------------------------- plain forms ----
def _ln_fwd(x, gamma, beta, dtype):
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = torch.rsqrt(c.square().mean(-1, keepdim=True) + LN_EPS)
    return {'y': (c * rstd * gamma + beta).to(dtype), 'mean': mean[:, 0], 'rstd': rstd[:, 0]}


def _ln_bwd(s):
    dy, rstd = s['dy'].float(), s['rstd'][:, None]
    xh = (s['x'].float() - s['mean'][:, None]) * rstd
    t = dy * s['gamma']
    dx = rstd * (t - t.mean(-1, keepdim=True) - xh * (t * xh).mean(-1, keepdim=True))
    if s['addend'] is not None:
        dx = dx + s['addend'].float()
    return {'dx': dx.to(s['x'].dtype), 'dgamma': (dy * xh).sum(0), 'dbeta': dy.sum(0)}


def _order(x):
    """int64 keys: larger value first, then lower index"""
    bits = (x + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7fffffff, bits).to(torch.int64)
    return bits * (1 << 32) + torch.arange(x.shape[1] - 1, -1, -1, device=x.device)


def _lp_parts(s):
    x, at = s['x'].float(), s['targets']
    m = x.max(-1, keepdim=True).values
    empty = m == -math.inf
    z = x - torch.where(empty, torch.zeros_like(m), m)
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    log_total = torch.where(empty, torch.full_like(m, -math.inf), total.log())
    lse = torch.where(empty, m, m + log_total)
    weighted = torch.where(e > 0, z * e, torch.zeros_like(z)).sum(-1, keepdim=True)
    entropy = torch.where(empty, torch.zeros_like(m), log_total - weighted / total)
    logp = z.gather(1, at.clamp(min=0)[:, None]) - torch.where(empty, torch.zeros_like(m), log_total)
    logp = torch.where(at[:, None] < 0, torch.zeros_like(logp), logp)
    k = _top(s['case'])
    index = torch.topk(_order(x), k, dim=-1).indices if k else None
    top = z.gather(1, index) - torch.where(empty, torch.zeros_like(m), log_total) if k else None
    return x, z, empty, log_total, {'logp': logp[:, 0], 'entropy': entropy[:, 0], 'lse': lse[:, 0], 'top': top, 'index': index}


def _lp_fwd(s):
    return _lp_parts(s)[-1]


def _lp_train(s):
    x, z, empty, log_total, got = _lp_parts(s)
    lp = z - torch.where(empty, torch.zeros_like(log_total), log_total)
    p = torch.where(empty, torch.zeros_like(z), torch.exp(lp))
    g = torch.where(s['targets'] < 0, torch.zeros_like(s['g_logp']), s['g_logp'])[:, None]
    total = g if got['index'] is None else g + s['g_top'].sum(-1, keepdim=True)
    gh = s['g_entropy'][:, None]
    dx = -total * p - torch.where(p > 0, gh * p * (lp + got['entropy'][:, None]), torch.zeros_like(p))
    dx.scatter_add_(1, s['targets'].clamp(min=0)[:, None], g)
    if got['index'] is not None:
        dx.scatter_add_(1, got['index'], s['g_top'])
    dx = torch.where(empty, torch.zeros_like(dx), dx)
    return {'logp': got['logp'], 'entropy': got['entropy'], 'top': got['top'], 'index': got['index'],
            'dx': dx.to(s['x'].dtype)}


def _groups(mats):
    found = {}
    for i, u in enumerate(mats):
        found.setdefault(tuple(u.shape), []).append(i)
    return found


def _orthogonal(mats):
    """Newton-Schulz on each matrix; those of one shape go through the products together"""
    a, b, c = COEF
    out = [None] * len(mats)
    for (rows, cols), at in _groups(mats).items():
        x = torch.stack([mats[i] for i in at])
        x = x.transpose(1, 2).contiguous() if rows > cols else x
        x = x / torch.sqrt(x.double().square().sum((1, 2), keepdim=True)).float().clamp(min=NS_EPS)
        for _ in range(NS_STEPS):
            gram = torch.matmul(x, x.transpose(1, 2))
            x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
        x = x.transpose(1, 2) if rows > cols else x
        for k, i in enumerate(at):
            out[i] = x[k].contiguous()
    return out


def _muon(s):
    u = []
    for w, v, g in zip(s['w'], s['v'], s['g']):
        g = g + WD * w
        v.mul_(MU).add_(g)
        u.append(g + MU * v if s['case']['nesterov'] else v)
    for w, o in zip(s['w'], _orthogonal(u)):
        w.sub_(o * (LR * _scale(*o.shape)))
    return {'w': s['flat_w'], 'v': s['flat_v']}


# ---------------------------------------------------------------- the definitions, 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    if op in ('ln_fwd', 'ln_bwd'):
        x, gamma, beta = s['x'].double(), s['gamma'].double(), s['beta'].double()
        if op == 'ln_fwd':
            var, mu = torch.var_mean(x, dim=1, unbiased=False)
            y = (x - mu[:, None]) / torch.sqrt(var + LN_EPS)[:, None] * gamma[None] + beta[None]
            return {'y': y, 'mean': mu, 'rstd': (var + LN_EPS) ** -0.5}
        dy = s['dy'].double()
        hat = (x - s['mean'].double()[:, None]) * s['rstd'].double()[:, None]
        n = x.shape[1]
        t = dy * gamma[None]
        dx = (n * t - t.sum(1, keepdim=True) - hat * (t * hat).sum(1, keepdim=True)) * (s['rstd'].double() / n)[:, None]
        if s['addend'] is not None:
            dx += s['addend'].double()
        return {'dx': dx, 'dgamma': torch.einsum('rc,rc->c', dy, hat), 'dbeta': dy.sum(0)}
    if op in ('lp_fwd', 'lp_train'):
        return _exact_lp(s, case)
    if op == 'orth':
        return [_exact_ns(u.double()) for u in s['mats']]
    new_w, new_v = [], []
    for w, v, g in zip(s['w'], s['v'], s['g']):
        g = g.double() + WD * w.double()
        v = MU * v.double() + g
        o = _exact_ns(g + MU * v if case['nesterov'] else v)
        new_w.append((w.double() - LR * _scale(*w.shape) * o).reshape(-1))
        new_v.append(v.reshape(-1))
    return {'w': torch.cat(new_w), 'v': torch.cat(new_v)}


def _exact_ns(u):
    """One matrix, taken from the side that makes the Gram matrix small"""
    a, b, c = COEF
    x = u / max(float(torch.linalg.norm(u)), NS_EPS)
    tall = x.shape[0] > x.shape[1]
    for _ in range(NS_STEPS):
        if tall:
            g = x.t().contiguous() @ x
            x = a * x + x @ (b * g + c * (g @ g))
        else:
            g = x @ x.t().contiguous()
            x = a * x + (b * g + c * (g @ g)) @ x
    return x


def _exact_lp(s, case):
    rows, k = case['rows'], _top(case)
    out = {'logp': [], 'entropy': [], 'lse': [], 'top': [], 'index': None, 'dx': []}
    step = max(1, 40000000 // case['cols'])
    for lo in range(0, rows, step):
        x, at = s['x'][lo:lo + step].double(), s['targets'][lo:lo + step]
        lse = torch.logsumexp(x, 1)
        none = torch.isinf(lse)
        lp = torch.where(none[:, None], torch.full_like(x, -math.inf), x - lse[:, None])
        p = lp.exp()
        plogp = torch.where(p > 0, p * lp, torch.zeros_like(p))
        h = -plogp.sum(1)
        asked = at >= 0
        out['lse'].append(lse)
        out['entropy'].append(h)
        out['logp'].append(torch.where(asked, lp.gather(1, at.clamp(min=0)[:, None])[:, 0], torch.zeros_like(lse)))
        best = torch.sort(lp, dim=1, descending=True, stable=True) if k else None
        if k:
            out['top'].append(best.values[:, :k])
        if case['op'] == 'lp_train':
            g = torch.where(asked, s['g_logp'][lo:lo + step].double(), torch.zeros_like(lse))
            dx = -g[:, None] * p - s['g_entropy'][lo:lo + step].double()[:, None] * (plogp + p * h[:, None])
            dx[torch.arange(len(x), device=x.device), at.clamp(min=0)] += g
            if k:
                gt = s['g_top'][lo:lo + step].double()
                dx -= gt.sum(1, keepdim=True) * p
                dx.scatter_add_(1, best.indices[:, :k], gt)
            dx[none] = 0
            out['dx'].append(dx)
    out = {key: torch.cat(v) if v else None for key, v in out.items()}
    if case['op'] == 'lp_fwd':
        del out['dx']
    else:
        del out['lse']
    return out


def work(case):
    op, size = case['op'], SIZE[case['type']]
    if op in ('ln_fwd', 'ln_bwd'):
        n, d = case['rows'], case['cols']
        if op == 'ln_fwd':
            return {'bytes': 2 * n * d * size + 8 * n + 8 * d, 'flops': 8 * n * d}
        return {'bytes': (3 + case['addend']) * n * d * size + 8 * n + 12 * d, 'flops': 14 * n * d}
    if op in ('lp_fwd', 'lp_train'):
        n, v, k = case['rows'], case['cols'], _top(case)
        if op == 'lp_fwd':
            return {'bytes': n * v * size + n * (20 + 12 * k), 'flops': 6 * n * v}
        # the gradient needs the row's sum first: the logits are read for it once more
        return {'bytes': 3 * n * v * size + n * (24 + 16 * k), 'flops': 14 * n * v}
    # symmetric products are counted once; muon reads g, v, w and writes v, w
    flops = values = 0
    for rows, cols, count in _shapes(case['matrices']):
        m, n = min(rows, cols), max(rows, cols)
        flops += count * NS_STEPS * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)
        values += count * rows * cols
    return {'bytes': values * (2 * size if op == 'orth' else 20), 'flops': flops}
