"""Log probabilities, entropy, alternatives and their gradient (kernels.log_probs_fwd / _bwd, autograd.log_probs) against the
formulas in float64.

Tolerances, u = 2^-24, z = x - max: x - max rounds to |z| u; an exponential is off by 2 |z| u (its argument's product) and 4 u of its
own; a sum of up to 16384 classes rounds 64 times in a thread, some 10 times across, and once per segment when joined, so
log S is off by at most (100 + 4 E|z|) u, E = mean under p.  (Several segments in a thread round as often as that many parts
joined; a thread's maximum grows at most that often, by a factor with the errors of one exponential.)  The entropy's second sum has the same errors times |z|."""
import math

import pytest
import torch

from luminoth_amd import autograd as A
from luminoth_amd import kernels as K

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(rows, C, dtype, seed=0, scale=3.0, pad=0):
    g = torch.Generator().manual_seed(seed + 31 * rows + C)
    return (torch.randn((rows, C + pad), generator=g) * scale).to(dtype), torch.randint(0, C, (rows,), generator=g)


def reference(x, targets, k):
    """float64: logp, entropy, lse, top, index and the rows' E|z|, E z^2"""
    x = x.double()
    top = x.amax(-1, keepdim=True)
    empty = top[:, 0] == -math.inf
    z = x - torch.where(empty[:, None], torch.zeros_like(top), top)
    log_s = z.exp().sum(-1).log()                        # x - (top + log_s) would lose log_s in a row of the type's lowest value
    lse = torch.where(empty, top[:, 0], top[:, 0] + log_s)
    lp = torch.where(empty[:, None], torch.full_like(x, -math.inf), z - log_s[:, None])
    p = lp.exp()
    z = torch.where(p > 0, x - x.amax(-1, keepdim=True), torch.zeros_like(x))
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    logp = None
    if targets is not None:
        logp = lp.gather(1, targets.clamp(min=0)[:, None])[:, 0]
        logp = torch.where(targets < 0, torch.zeros_like(logp), logp)
    order = torch.sort(x + 0.0, dim=-1, descending=True, stable=True).indices[:, :k]
    return logp, -plp.sum(-1) + 0.0, lse, lp.gather(1, order), order, (p * z.abs()).sum(-1), (p * z * z).sum(-1), p, lp


def near(got, want, tol, what):
    got, want = got.cpu().double(), want
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    bad = ~same & ~((got - want).abs() <= tol)
    assert not bad.any(), (what, got[bad][:4], want[bad][:4], tol.expand_as(want)[bad][:4])


def check_fwd(x, targets, k, got):
    logp, entropy, top, index, lse = got
    rl, rh, rs, rt, ri, ez, ezz, _, _ = reference(x, targets, k)
    log_tol = (100 + 4 * ez) * U
    if targets is not None:
        near(logp, rl, log_tol + 3 * U * torch.where(torch.isfinite(rl), rl.abs(), torch.zeros_like(rl)), 'logp')
    else:
        assert logp is None
    near(lse, rs, log_tol + 2 * U * torch.where(torch.isfinite(rs), rs.abs(), torch.zeros_like(rs)), 'lse')
    near(entropy, rh, log_tol + (110 * ez + 4 * ezz) * U, 'entropy')
    if k:
        assert torch.equal(index.cpu(), ri), 'alternatives'
        near(top, rt, log_tol[:, None] + 3 * U * torch.where(torch.isfinite(rt), rt.abs(), torch.zeros_like(rt)), 'top')
    else:
        assert top is None and index is None


SHAPES = [(1, 1, 1), (2, 2, 2), (5, 21, 5), (7, 81, 64), (130, 81, 1), (3, 513, 20), (4, 1024, 3), (3, 1025, 64), (6, 2048, 20),
          (2, 5000, 33), (9, 16384, 5), (3, 16389, 7), (600, 4099, 2), (2, 70001, 20), (1, 131072, 20), (40, 40000, 0)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,C,k', SHAPES)
def test_forward(rows, C, k, dtype):
    x, t = make(rows, C, dtype)
    if rows > 2:
        t[1] = -1
    check_fwd(x, t, k, K.log_probs_fwd(x.cuda(), t.cuda(), k))
    check_fwd(x, None, k, K.log_probs_fwd(x.cuda(), None, k))
    check_fwd(x, t, 0, K.log_probs_fwd(x.cuda(), t.int().cuda(), 0))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('C', [100, 3000, 40000])
def test_ties_and_signed_zeros(C, dtype):
    """Few distinct values (every list overflows), rows of one value, zeros of both signs: the lowest index first."""
    g = torch.Generator().manual_seed(C)
    x = torch.randint(-2, 3, (6, C), generator=g).to(dtype)
    x[1] = 0.5
    x[2] = 0.0
    x[2, ::2] = -0.0
    x[3] = torch.linspace(-9, 9, C).to(dtype)             # ascending: the large ones in few lanes
    x[4] = torch.linspace(9, -9, C).to(dtype)
    for k in (1, 20, 64):
        check_fwd(x, torch.zeros(6, dtype=torch.int64), k, K.log_probs_fwd(x.cuda(), torch.zeros(6, dtype=torch.int64).cuda(), k))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('C', [90, 5000, 33333])
def test_masks(C, dtype):
    """Classes of -inf and of the type's lowest value; rows with one class left, with none, with fewer than k."""
    x, t = make(8, C, dtype)
    low = torch.finfo(dtype).min
    x[0, 1:] = -math.inf
    x[1] = -math.inf
    x[2, torch.arange(C) % 7 != 3] = -math.inf
    x[3, 5:] = low
    x[4] = low
    x[5, : C - 10] = -math.inf
    x[6, C // 2:] = -math.inf
    t[0], t[1], t[5] = 0, 2, 0
    check_fwd(x, t, 20, K.log_probs_fwd(x.cuda(), t.cuda(), 20))
    logp, entropy, top, index, lse = (v.cpu() for v in K.log_probs_fwd(x.cuda(), t.cuda(), 20))
    assert logp[0] == 0 and entropy[0] == 0 and logp[1] == -math.inf and entropy[1] == 0 and lse[1] == -math.inf
    assert torch.equal(index[1], torch.arange(20)) and (top[1] == -math.inf).all() and logp[5] == -math.inf


@pytest.mark.parametrize('rows,C,dtype', [(2100, 16389, torch.float32), (1400, 33001, torch.bfloat16), (4200, 16390, torch.float16)])
@pytest.mark.parametrize('k', [1, 20, 40])
def test_many_rows(rows, C, dtype, k):
    """Enough rows that a block takes several segments of one: ordinary rows, rows in order, of one value, of few values, masked
    ones.  The reference runs on the GPU in float64, on every 7th row and those."""
    g = torch.Generator(device='cuda').manual_seed(C)
    x = (torch.randn((rows, C), generator=g, device='cuda') * 3).to(dtype)
    t = torch.randint(0, C, (rows,), generator=g, device='cuda')
    x[0] = torch.linspace(-9, 9, C, device='cuda')
    x[7] = torch.linspace(9, -9, C, device='cuda')
    x[14] = 1.5
    x[21] = torch.randint(-3, 3, (C,), generator=g, device='cuda').to(dtype)
    x[28] = -math.inf
    x[35, torch.randperm(C, generator=g, device='cuda')[: C - 9]] = -math.inf
    x[42, : C - 5] = -math.inf
    x[49, 11:] = -math.inf
    x[56, ::2] = -math.inf
    x[63] = 0.0
    x[63, ::3] = -0.0
    x[70, C // 2] = math.nan
    t[77] = -1
    got = K.log_probs_fwd(x, t, k)
    at = torch.arange(0, rows, 7)
    at = at[at != 70]
    xs = x[at.cuda()].cpu()
    check_fwd(xs, t[at.cuda()].cpu(), k, [v[at.cuda()].cpu() for v in got])
    assert torch.isnan(got[0][70]) and torch.isnan(got[2][70]).all() and int(got[3][70, 0]) == C // 2
    other = K.log_probs_fwd(x, t, 0)                       # without alternatives: the same sums
    for a, b in zip(got, other):
        if b is not None:
            assert torch.equal(a.nan_to_num(7), b.nan_to_num(7)) or k > 32


@pytest.mark.parametrize('rows,C,dtype,k', [(2, 1000003, torch.float32, 40), (2, 300007, torch.bfloat16, 64), (3000, 20000, torch.float16, 64)])
def test_long_lists_of_alternatives(rows, C, dtype, k):
    """More vectors than the list of a part holds, and more parts than 64."""
    g = torch.Generator(device='cuda').manual_seed(k)
    x = (torch.randn((rows, C), generator=g, device='cuda') * 2).to(dtype)
    x[0] = torch.linspace(-20, 20, C, device='cuda')
    x[1, 5:] = x[1, 5]
    t = torch.arange(rows, device='cuda')
    got = K.log_probs_fwd(x, t, k)
    n = min(rows, 200)
    check_fwd(x[:n].cpu(), t[:n].cpu(), k, [v[:n].cpu() for v in got])


def test_not_a_number_and_no_class():
    x, t = make(5, 3000, torch.float32)
    x[1, 17] = math.nan
    x[2, 40] = math.inf
    t[3], t[4] = 3000, 2 ** 40
    logp, entropy, top, index, lse = (v.cpu() for v in K.log_probs_fwd(x.cuda(), t.cuda(), 4))
    assert torch.isnan(logp[1:]).all() and torch.isnan(entropy[1:3]).all() and torch.isnan(lse[1:3]).all()
    assert torch.isnan(top[1:3]).all() and index[1, 0] == 17 and index[2, 0] == 40
    check_fwd(x[:1], t[:1], 4, [v[:1] for v in (logp, entropy, top, index, lse)])
    assert torch.isfinite(entropy[3:]).all()
    out = K.log_probs_fwd(torch.empty((0, 9), device='cuda'), torch.empty((0,), dtype=torch.int64, device='cuda'), 2)
    assert out[0].shape == (0,) and out[2].shape == (0, 2) and out[3].dtype == torch.int64
    assert K.log_probs_bwd(torch.empty((0, 9), device='cuda'), None, out[4], out[1], g_entropy=out[1]).shape == (0, 9)


@pytest.mark.parametrize('dtype', TYPES)
def test_rows_of_a_padded_buffer(dtype):
    full, _ = make(11, 2500, dtype, pad=13)
    t = torch.arange(11) * 200
    x = full.cuda()
    x[:, 2500:] = 99.0                                     # behind the classes: never looked at
    check_fwd(full[:, :2500], t, 9, K.log_probs_fwd(x[:, :2500], t.cuda(), 9))
    lead = K.log_probs_fwd(full.cuda()[:, 1:2401].unflatten(0, (1, 11)), t.cuda()[None], 9)
    assert lead[0].shape == (1, 11) and lead[2].shape == (1, 11, 9)
    check_fwd(full[:, 1:2401], t, 9, [v[0] for v in lead])


def bwd_reference(x, targets, gl, gh, index, gt):
    _, h, lse, _, _, ez, ezz, p, lp = reference(x, targets, 0)
    g = torch.zeros(len(x), dtype=torch.float64) if gl is None else torch.where(targets < 0, 0.0, gl.double())
    total = g if gt is None else g + gt.double().sum(-1)
    lp0 = torch.where(p > 0, lp, torch.zeros_like(lp))
    dx = -total[:, None] * p
    if gh is not None:
        dx = dx - gh.double()[:, None] * p * (lp0 + h[:, None])
    own = torch.zeros_like(dx)
    if gl is not None:
        own.scatter_add_(1, targets.clamp(min=0)[:, None], g[:, None])
    if gt is not None:
        own.scatter_add_(1, index, gt.double())
    dx = torch.where((lse == -math.inf)[:, None], torch.zeros_like(dx), dx + own)
    # p: the row's log sum, x - lse and the exponential
    rel = (120 + 4 * ez + 2 * torch.where(torch.isfinite(lse), lse.abs(), torch.zeros_like(lse)))[:, None] + 6 * lp0.abs()
    size = total.abs()[:, None] + (0 if gt is None else 64 * gt.double().abs().sum(-1, keepdim=True) * U)
    if gh is not None:
        size = size + gh.double().abs()[:, None] * (lp0.abs() + h[:, None] + 2 + (120 * ez + 4 * ezz)[:, None] * U + 1)
    tol = U * (rel * p * size + 70 * own.abs() + (0 if gt is None else 70 * gt.double().abs().sum(-1, keepdim=True) * (own != 0)) +
               4 * dx.abs())
    return dx, tol


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,C,k', [(1, 1, 1), (3, 2, 2), (7, 81, 5), (5, 1030, 20), (4, 9001, 64), (300, 2048, 3), (2, 70001, 8)])
def test_backward(rows, C, k, dtype):
    x, t = make(rows, C, dtype, seed=4)
    if rows > 2:
        t[1] = -1
        x[2, C // 2:] = -math.inf
        t[2] = 0
    if rows > 3:
        x[3] = -math.inf
    g = torch.Generator().manual_seed(k)
    gl, gh, gt = torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn((rows, k), generator=g)
    logp, entropy, top, index, lse = K.log_probs_fwd(x.cuda(), t.cuda(), k)
    for use in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
        a, b, c = (v if u else None for u, v in zip(use, (gl, gh, gt)))
        dx = K.log_probs_bwd(x.cuda(), t.cuda(), lse, entropy, *(None if v is None else v.cuda() for v in (a, b)),
                             index if c is not None else None, None if c is None else c.cuda())
        want, tol = bwd_reference(x, t, a, b, index.cpu(), c)
        tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
        near(dx, want, tol, use)


def test_alternatives_given_twice():
    """The target among the alternatives and one alternative named three times: every gradient arrives."""
    x, _ = make(2, 500, torch.float32)
    t = torch.tensor([3, 4])
    index = torch.tensor([[3, 3, 9, 3], [7, 4, 7, 499]])
    gl, gt = torch.tensor([1.0, -2.0]), torch.tensor([[0.5, 0.25, 1.0, -3.0], [1.0, 2.0, 3.0, 4.0]])
    _, entropy, _, _, lse = K.log_probs_fwd(x.cuda(), None, 0)
    dx = K.log_probs_bwd(x.cuda(), t.cuda(), lse, entropy, gl.cuda(), None, index.cuda(), gt.cuda())
    want, tol = bwd_reference(x, t, gl, None, index, gt)
    near(dx, want, tol + U * want.abs(), 'twice')


def test_gradient_against_differences():
    g = torch.Generator().manual_seed(0)
    x = torch.randn((3, 40), generator=g) * 2
    t = torch.tensor([5, -1, 39])
    a, b, c = torch.randn(3, generator=g), torch.randn(3, generator=g), torch.randn((3, 4), generator=g)
    leaf = x.cuda().requires_grad_()
    logp, entropy, top, index = A.log_probs(leaf, t.cuda(), 4)
    assert not index.requires_grad
    ((logp * a.cuda()).sum() + (entropy * b.cuda()).sum() + (top * c.cuda()).sum()).backward()
    order = index.cpu()

    def f(v):
        lp = torch.log_softmax(v, -1)
        s = (torch.where(t < 0, 0.0, lp.gather(1, t.clamp(min=0)[:, None])[:, 0]) * a.double()).sum()
        return s - ((lp.exp() * lp).sum(-1) * b.double()).sum() + (lp.gather(1, order) * c.double()).sum()
    h = 1e-5
    base = x.double()
    flat = base.view(-1)
    for i in range(0, 120, 7):
        v = float(flat[i])
        flat[i] = v + h
        up = f(base)
        flat[i] = v - h
        down = f(base)
        flat[i] = v
        # a central difference is off by h^2 f''' / 6 (below 1e-9 here) and 1e-16 / h
        assert abs(float(leaf.grad.view(-1)[i]) - float(up - down) / (2 * h)) <= 2e-5


def test_gradients_of_some_outputs_only():
    x, t = make(4, 300, torch.bfloat16)
    leaf = x.cuda().requires_grad_()
    logp, _, _, _ = A.log_probs(leaf, t.cuda())
    logp.sum().backward()                                  # (an expanded gradient)
    want, tol = bwd_reference(x, t, torch.ones(4), None, None, None)
    near(leaf.grad, want, tol + 2.0 ** -8 * want.abs() + 1e-37, 'logp alone')
    _, entropy, top, index = A.log_probs(leaf, None, 2)
    assert torch.autograd.grad(entropy.sum(), leaf)[0].shape == leaf.shape


def test_streams_and_graph():
    x, t = make(9, 30000, torch.bfloat16)
    x, t = x.cuda(), t.cuda()
    want = K.log_probs_fwd(x, t, 6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.log_probs_fwd(x, t, 6)
    with K.launch_on(side):
        again = K.log_probs_fwd(x, t, 6)
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, again):
        assert torch.equal(a, b) and torch.equal(a, c)
    ones = torch.ones(9, device='cuda')
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logp, entropy, top, index, lse = K.log_probs_fwd(x, t, 6)
        dx = K.log_probs_bwd(x, t, lse, entropy, ones, ones)
    for seed in range(4):
        x.copy_(make(9, 30000, torch.bfloat16, seed=seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        e = K.log_probs_fwd(x, t, 6)
        for a, b in zip((logp, entropy, top, index, lse, dx), e + (K.log_probs_bwd(x, t, e[4], e[1], ones, ones),)):
            assert torch.equal(a, b)


@pytest.mark.parametrize('C', [20, 3000])
def test_targets_of_32_bits_and_repeated_alternatives(C):
    x, t = make(7, C, torch.bfloat16)
    t[2] = -1
    dev, t64, t32 = x.cuda(), t.cuda(), t.int().cuda()
    for a, b in zip(K.log_probs_fwd(dev, t64, 3), K.log_probs_fwd(dev, t32, 3)):
        assert torch.equal(a, b)
    _, entropy, _, _, lse = K.log_probs_fwd(dev, None, 0)
    index = torch.tensor([[C - 1, 0, C - 1, 5]] * 7)
    gl, gt = torch.linspace(-1, 1, 7), torch.linspace(-3, 2, 28).view(7, 4)
    dx = [K.log_probs_bwd(dev, v, lse, entropy, gl.cuda(), None, index.cuda(), gt.cuda()) for v in (t64, t32)]
    assert torch.equal(dx[0], dx[1])
    want, tol = bwd_reference(x, t, gl, None, index, gt)
    near(dx[0], want, tol + 2.0 ** -8 * (want.abs() + tol) + 1e-37, 'repeated')


def test_rows_far_apart_and_results_beyond_32_bits():
    ld, t = 2 ** 30 + 64, torch.tensor([5, 2999, 0]).cuda()
    far = torch.empty(3 * ld, device='cuda', dtype=torch.bfloat16)
    x = far.as_strided((3, 3000), (ld, 1))
    x.copy_(make(3, 3000, torch.bfloat16)[0])
    got, want = K.log_probs_fwd(x, t, 4), K.log_probs_fwd(x.contiguous(), t, 4)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    ones = torch.ones(3, device='cuda')
    assert torch.equal(K.log_probs_bwd(x, t, got[4], got[1], ones, ones), K.log_probs_bwd(x.contiguous(), t, got[4], got[1], ones, ones))
    del far, x
    rows, C = 2 ** 16 + 3, 33000
    x = torch.empty((rows, C), device='cuda', dtype=torch.bfloat16).normal_()
    t = torch.randint(0, C, (rows,), generator=torch.Generator().manual_seed(0))
    logp, entropy, top, index, lse = K.log_probs_fwd(x, t.cuda(), 2)
    check_fwd(x[-3:].cpu(), t[-3:], 2, [v[-3:] for v in (logp, entropy, top, index, lse)])
    ones = torch.ones(rows, device='cuda')
    dx = K.log_probs_bwd(x, t.cuda(), lse, entropy, ones, ones)
    want, tol = bwd_reference(x[-3:].cpu(), t[-3:], torch.ones(3), torch.ones(3), None, None)
    near(dx[-3:], want, tol + 2.0 ** -8 * (want.abs() + tol) + 1e-37, 'last rows')


def test_two_graphs_in_turn():
    """Two captured calls whose rows are joined from parts, replayed one behind the other with eager calls between."""
    inputs, graphs, outs = [], [], []
    for seed, C in ((0, 300007), (1, 70001)):
        x, t = make(3, C, torch.float32, seed=seed)
        inputs.append((x.cuda(), t.cuda(), 5))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(K.log_probs_fwd(*inputs[-1]))
        graphs.append(graph)
    for _ in range(3):
        for x, _, _ in inputs:
            x.mul_(-0.75)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for args, got in zip(inputs, outs):
            for a, b in zip(got, K.log_probs_fwd(*args)):
                assert torch.equal(a, b)
