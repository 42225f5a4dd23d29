"""The gradient of log probabilities (kernels.log_probs_bwd, autograd.log_probs) for logits far from zero, against float64: softmax does
not change when a constant is added to a row, and neither does what its gradient is off by.

Tolerances, u = 2^-24, z = x - max: as in test_gpu_log_probs.py the log of a row's sum is off by at most (100 + 4 E|z|) u, in the forward
pass and once more where the backward sums exp(x - lse); there each exponential is off by 3 |x - lse| u + 4 u, E|x - lse| <= E|z| + log S; an
entry's exponential by 3 |log p| u + 4 u.  Below |lse| = 32 the gradient takes lse as it was rounded: |lse| u.  Nothing grows with
the offset beyond."""
import math

import pytest
import torch

from luminoth_amd import autograd as A
from luminoth_amd import kernels as K

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SHAPES = [(5, 21), (9, 81), (3, 1024), (4, 1030), (6, 5000), (40, 16389), (2, 70001), (300, 3000), (1300, 9001)]


def reference(x, t, gl, gh, index, gt):
    """float64 -> dx and what it may be off by before its rounding to x's type"""
    x = x.double()
    z = x - x.amax(-1, keepdim=True)
    log_s = z.exp().sum(-1, keepdim=True).log()
    lp = z - log_s
    p = lp.exp()
    lp0, z0 = (torch.where(p > 0, v, torch.zeros_like(v)) for v in (lp, z))
    h, ez, ezz = -(p * lp0).sum(-1, keepdim=True), (p * z0.abs()).sum(-1, keepdim=True), (p * z0 * z0).sum(-1, keepdim=True)
    own = torch.zeros_like(x).scatter_add_(1, t[:, None], gl.double()[:, None]).scatter_add_(1, index, gt.double())
    G, gh = (gl.double() + gt.double().sum(-1))[:, None], gh.double()[:, None]
    dx = own - p * (G + gh * (lp0 + h))
    lse = x.amax(-1, keepdim=True) + log_s
    rel = 240 + 11 * ez + 3 * log_s + torch.where(lse.abs() < 40, lse.abs(), torch.zeros_like(lse)) + 6 * lp0.abs()
    given = gl.double().abs()[:, None] + gt.double().abs().sum(-1, keepdim=True)
    size = G.abs() + gh.abs() * (lp0.abs() + h + 1)
    tol = U * (p * (rel * size + gh.abs() * (rel + 110 * ez + 4 * ezz) + 70 * given) + 70 * given * (own != 0) + 4 * dx.abs())
    return dx, tol


def gradients(rows, k, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn((rows, k), generator=g)


def check(dx, x, want, tol):
    half = torch.finfo(x.dtype).eps / 2
    tol = tol + half * (want.abs() + tol) + (2.0 ** -25 if x.dtype == torch.float16 else 1e-37)
    err = (dx.cpu().double() - want).abs()
    assert (err <= tol).all(), (float(err.max()), float((err / tol).max()))
    # sum over the classes of own - p (G + ...) is zero: what is left is what the entries may be off by
    assert (dx.cpu().double().sum(-1).abs() <= tol.sum(-1)).all()


@pytest.mark.parametrize('dtype,offset', [(torch.float32, o) for o in (30.0, -37.0, 1e2, -1e3, 1e4, 1e5, -1e6)] +
                         [(torch.float16, o) for o in (-200.0, 3e4)] + [(torch.bfloat16, o) for o in (60.0, -1e4)])
@pytest.mark.parametrize('rows,C', SHAPES)
def test_logits_around_an_offset(rows, C, dtype, offset):
    g = torch.Generator().manual_seed(rows + C)
    x = (torch.randn((rows, C), generator=g) * 3 + offset).to(dtype)
    if rows > 3:
        x[3, C // 3:] = -math.inf
        x[2] += offset / 2 if dtype == torch.float32 else 0          # another offset beside it
    t = torch.randint(0, max(1, C // 3), (rows,), generator=g)
    k = 3
    gl, gh, gt = gradients(rows, k, C)
    dev = x.cuda()
    logp, entropy, top, index, lse = K.log_probs_fwd(dev, t.cuda(), k)
    dx = K.log_probs_bwd(dev, t.cuda(), lse, entropy, gl.cuda(), gh.cuda(), index, gt.cuda())
    want, tol = reference(x, t, gl, gh, index.cpu(), gt)
    check(dx, x, want, tol)
    if dtype == torch.float32:
        leaf = dev.clone().requires_grad_()
        lp, h, tp, _ = A.log_probs(leaf, t.cuda(), k)
        ((lp * gl.cuda()).sum() + (h * gh.cuda()).sum() + (tp * gt.cuda()).sum()).backward()
        assert torch.equal(leaf.grad, dx)


def test_rows_near_and_far_in_a_padded_buffer():
    """Rows above and below the border in one call, rows of a wider buffer, a masked row, not-a-number, one that is infinite"""
    full = torch.randn((12, 5000 + 9), generator=torch.Generator().manual_seed(0)) * 2
    full += torch.tensor([0.0, 100.0, -100.0, 20.0, 24.0, 28.0, 40.0, 0.0, 1e30, -1e30, 0.0, 0.0])[:, None]
    x = full[:, :5000]
    x[7] = -math.inf
    x[10, 3] = math.nan
    x[11, 3] = math.inf
    t = torch.arange(12) * 7
    gl, gh, gt = gradients(12, 2, 1)
    dev = full.cuda()[:, :5000]
    _, entropy, _, index, lse = K.log_probs_fwd(dev, t.cuda(), 2)
    dx = K.log_probs_bwd(dev, t.cuda(), lse, entropy, gl.cuda(), gh.cuda(), index, gt.cuda())
    assert (dx[7] == 0).all() and torch.isnan(dx[10]).all() and torch.isnan(dx[11]).all()
    at = [0, 1, 2, 3, 4, 5, 6, 8, 9]
    want, tol = reference(x[at], t[at], gl[at], gh[at], index.cpu()[at], gt[at])
    check(dx[at], x, want, tol)


@pytest.mark.parametrize('C', [60, 40000])
def test_lse_of_more_classes_than_these(C):
    """Half of a vocabulary with the lse of all of it: p = exp(x - lse) as given, nothing is made to sum to one"""
    g = torch.Generator().manual_seed(C)
    x = (torch.randn((70, 2 * C), generator=g) + 500).cuda()
    lse = K.log_probs_fwd(x)[4]
    half, ones = x[:, :C], torch.ones(70, device='cuda')
    t = torch.zeros(70, dtype=torch.int64, device='cuda')
    dx = K.log_probs_bwd(half, t, lse, None, ones).cpu().double()
    want = -(half.cpu().double() - lse.cpu().double()[:, None]).exp()
    want[:, 0] += 1
    # x - lse is exact to an ulp of the difference here (below 16), the exponential to 3 |x - lse| u + 4 u
    assert (dx - want).abs().max() <= 60 * U


def test_graph_of_rows_far_from_zero():
    x = torch.randn((5, 20000), generator=torch.Generator().manual_seed(2)).cuda() + 3000
    ones, t = torch.ones(5, device='cuda'), torch.zeros(5, dtype=torch.int64, device='cuda')
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, h, _, _, lse = K.log_probs_fwd(x, t)
        dx = K.log_probs_bwd(x, t, lse, h, ones, ones)
    for _ in range(4):
        x.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        _, h2, _, _, l2 = K.log_probs_fwd(x, t)
        assert torch.equal(dx, K.log_probs_bwd(x, t, l2, h2, ones, ones)) and torch.isfinite(dx).all()
