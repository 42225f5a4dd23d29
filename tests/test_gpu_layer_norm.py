"""Layer norm (kernels.layer_norm_fwd / _bwd, autograd.layer_norm) against the formula in float64.

Tolerances: u = 2^-24 is half a step of float32.  A sum over D columns rounds at most 16 times inside a thread and 10 times
across threads (the long-row kernel: D / 4096 * 8 + 10 times), so a mean is off by at most N u mean|.| with N = that count + 2;
what is computed from it is a few roundings more.  The result is rounded once: half a step of its type, eps / 2 of the value."""
import math

import pytest
import torch

from luminoth_amd import autograd as A
from luminoth_amd import kernels as K

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def roundings(D):
    return (28 if D <= 16384 else 8 * (D // 4096 + 1) + 12)


def make(rows, D, dtype, pad=0, seed=0, offset=1.0):
    g = torch.Generator().manual_seed(seed + 7 * rows + D)
    full = torch.randn((rows, D + pad), generator=g) + offset * torch.randn((rows, 1), generator=g)
    return full.to(dtype)


def fwd_ref(x, gamma, beta, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    xh = (x - mean) * rstd
    y = xh if gamma is None else xh * gamma.double()
    return mean[..., 0], rstd[..., 0], xh, y if beta is None else y + beta.double()


def check_fwd(x, gamma, beta, eps, got, dtype):
    y, mean, rstd = (t.cpu().double() for t in got)
    D = x.shape[-1]
    N = roundings(D)
    rm, rr, xh, ry = fwd_ref(x, gamma, beta, eps)
    ax = x.double().abs()
    tol_mean = (N + 2) * U * ax.mean(-1)
    assert ((mean - rm).abs() <= tol_mean + 1e-37).all()
    # variance: its own sum, and the mean's error (first order: it cancels in the sum of the deviations; squared it is negligible)
    rel = (N + 8) * U + 2 * (tol_mean * rr) ** 2
    assert ((rstd - rr).abs() <= rel * rr).all()
    g = 1.0 if gamma is None else gamma.double().abs()
    tol = g * (xh.abs() * (rel + 6 * U)[..., None] + (rr * (tol_mean + U * ax.amax(-1)))[..., None]) + 2 * U * ry.abs()
    tol = tol + torch.finfo(dtype).eps / 2 * (ry.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0)
    bad = (y - ry).abs() > tol
    assert not bad.any(), ((y - ry).abs() / tol).max()


def run_fwd(x, gamma, beta, eps=1e-5):
    dev = lambda t: None if t is None else t.cuda()      # noqa: E731
    return K.layer_norm_fwd(x, dev(gamma), dev(beta), eps)


SHAPES = [(1, 1), (3, 2), (5, 7), (17, 32), (65, 81), (4, 255), (4, 257), (9, 1000), (130, 1024), (7, 1025), (33, 4096), (5, 4097),
          (3, 16384), (3, 16385), (2, 40003), (1, 8192), (700, 64), (2049, 33)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,D', SHAPES)
def test_forward(rows, D, dtype):
    x = make(rows, D, dtype)
    g = torch.Generator().manual_seed(1)
    gamma, beta = 1 + torch.randn(D, generator=g) * 0.3, torch.randn(D, generator=g)
    check_fwd(x, gamma, beta, 1e-5, run_fwd(x.cuda(), gamma, beta), dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('pad,skip', [(1, 0), (5, 3), (64, 0)])
def test_rows_of_a_wider_buffer(dtype, pad, skip):
    full = make(19, 200 + pad, dtype)
    x = full.cuda()[:, skip:skip + 200]
    assert not x.is_contiguous()
    check_fwd(full[:, skip:skip + 200], None, None, 1e-5, run_fwd(x, None, None), dtype)


def test_leading_dimensions_parameters_and_offsets():
    x = make(24, 96, torch.bfloat16, offset=20.0)
    g = torch.Generator().manual_seed(2)
    gamma, beta = (1 + torch.randn(96, generator=g)).bfloat16(), torch.randn(96, generator=g).bfloat16()
    y, mean, rstd = run_fwd(x.view(2, 3, 4, 96).cuda(), gamma, beta)
    assert y.shape == (2, 3, 4, 96) and mean.shape == (2, 3, 4) and rstd.dtype == torch.float32
    check_fwd(x, gamma, beta, 1e-5, (y.view(24, 96), mean.view(24), rstd.view(24)), torch.bfloat16)
    check_fwd(x, gamma, None, 1e-3, run_fwd(x.cuda(), gamma, None, 1e-3), torch.bfloat16)
    check_fwd(x, None, beta, 1e-5, run_fwd(x.cuda(), None, beta), torch.bfloat16)


def test_constant_rows_infinities_and_no_rows():
    x = torch.full((4, 50), 3.25)
    x[1] = 0
    x[2, 7] = math.inf
    x[3, 0] = math.nan
    y, mean, rstd = K.layer_norm_fwd(x.cuda())
    assert (y[:2] == 0).all() and torch.isnan(y[2:]).all()
    assert torch.allclose(rstd[:2].cpu(), torch.full((2,), 1e-5 ** -0.5), rtol=1e-6)
    y, mean, rstd = K.layer_norm_fwd(torch.empty((0, 5), device='cuda'))
    assert y.shape == (0, 5) and mean.shape == (0,)
    dg, db = torch.full((5,), 7.0, device='cuda'), torch.full((5,), 7.0, device='cuda')
    dx = K.layer_norm_bwd(y, y, mean, rstd, None, dg, db)
    assert dx.shape == (0, 5) and (dg == 0).all() and (db == 0).all()


def bwd_ref(dy, x, mean, rstd, gamma, addend):
    dy, xh = dy.double(), (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    t = dy if gamma is None else dy * gamma.double()
    a, b = t.mean(-1, keepdim=True), (t * xh).mean(-1, keepdim=True)
    dx = rstd.double()[:, None] * (t - a - xh * b)
    if addend is not None:
        dx = dx + addend.double()
    return dx, xh, t, a, b


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,D', SHAPES)
def test_backward(rows, D, dtype):
    x, dy = make(rows, D, dtype), make(rows, D, dtype, seed=5, offset=0.2)
    addend = make(rows, D, dtype, seed=9) if rows % 2 else None
    g = torch.Generator().manual_seed(1)
    gamma = 1 + torch.randn(D, generator=g) * 0.3
    mean, rstd = (t.float() for t in fwd_ref(x, None, None, 1e-5)[:2])
    dg, db = torch.full((D,), 9.0, device='cuda'), torch.full((D,), 9.0, device='cuda')
    dx = K.layer_norm_bwd(dy.cuda(), x.cuda(), mean.cuda(), rstd.cuda(), gamma.cuda(), dg, db,
                          addend=None if addend is None else addend.cuda())
    rx, xh, t, a, b = bwd_ref(dy, x, mean, rstd, gamma, addend)
    N = roundings(D) + 4
    at, axh = t.abs(), xh.abs() + U * (x.double().abs() * rstd.double()[:, None])
    tol = U * rstd.double()[:, None] * (6 * at + N * at.mean(-1, keepdim=True) + axh * N * (at * axh).mean(-1, keepdim=True) +
                                       6 * axh * b.abs() + 4 * a.abs())
    if addend is not None:
        tol = tol + U * rx.abs()
    tol = tol + torch.finfo(dtype).eps / 2 * (rx.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0) + 1e-37
    err = (dx.cpu().double() - rx).abs()
    assert not (err > tol).any(), (err / tol).max()
    # sums over the rows, in any order: at most one rounding per addition
    n = (rows + 40) * U
    for got, ref, size in ((dg, dy.double() * xh, (dy.double().abs() * axh)), (db, dy.double(), dy.double().abs())):
        err = (got.cpu().double() - ref.sum(0)).abs()
        assert not (err > (n + 4 * U) * size.sum(0) + 1e-37).any(), err.max()


@pytest.mark.parametrize('D', [48, 1024, 5000, 20000])
def test_what_the_backward_writes(D):
    """dx alone, the parameters alone, 16-bit parameters; the same bits every time; nothing behind the rows."""
    x, dy = make(37, D, torch.bfloat16).cuda(), make(37, D, torch.bfloat16, seed=3).cuda()
    gamma = (1 + 0.2 * torch.randn(D, generator=torch.Generator().manual_seed(0))).bfloat16().cuda()
    y, mean, rstd = K.layer_norm_fwd(x, gamma)
    dg, db = torch.empty(D, device='cuda', dtype=torch.bfloat16), torch.empty(D, device='cuda', dtype=torch.bfloat16)
    dx = K.layer_norm_bwd(dy, x, mean, rstd, gamma, dg, db)
    assert torch.equal(dx, K.layer_norm_bwd(dy, x, mean, rstd, gamma))
    dg2, db2 = torch.empty_like(dg), torch.empty_like(db)
    assert K.layer_norm_bwd(dy, x, mean, rstd, gamma, dg2, None, need_dx=False) is None
    assert torch.equal(dg, dg2)
    K.layer_norm_bwd(dy, x, mean, rstd, gamma, None, db2, need_dx=False)
    assert torch.equal(db, db2)
    for _ in range(3):
        dg2, db2 = torch.empty_like(dg), torch.empty_like(db)
        assert torch.equal(dx, K.layer_norm_bwd(dy, x, mean, rstd, gamma, dg2, db2))
        assert torch.equal(dg, dg2) and torch.equal(db, db2)


@pytest.mark.parametrize('D', [7, 130])
def test_gradient_against_differences(D):
    """autograd.layer_norm: central differences of sum(y * r) in float64 of the formula at the same point."""
    g = torch.Generator().manual_seed(D)
    x, r = torch.randn((5, D), generator=g), torch.randn((5, D), generator=g)
    gamma, beta = 1 + 0.3 * torch.randn(D, generator=g), torch.randn(D, generator=g)
    leaves = [t.cuda().requires_grad_() for t in (x, gamma, beta)]
    y = A.layer_norm(*leaves)
    (y * r.cuda()).sum().backward()

    def f(x, gamma, beta):
        return (fwd_ref(x, gamma, beta, 1e-5)[3] * r.double()).sum()
    h = 1e-5
    for k, leaf in enumerate(leaves):
        base = [x.double(), gamma.double(), beta.double()]
        flat = base[k].reshape(-1)
        for i in range(0, flat.numel(), max(1, flat.numel() // 11)):
            v = float(flat[i])
            flat[i] = v + h
            up = f(*base)
            flat[i] = v - h
            down = f(*base)
            flat[i] = v
            want = float(up - down) / (2 * h)
            # the difference's own error: h^2 times a third derivative of some units, and float32's
            assert abs(float(leaf.grad.reshape(-1)[i]) - want) <= 1e-5 * (1 + abs(want)) * D ** 0.5


def test_gradient_of_a_broadcast_result():
    """y.sum(): the gradient arrives as one value expanded to all of y; x alone needs a gradient."""
    x = make(6, 40, torch.float32).cuda().requires_grad_()
    A.layer_norm(x).sum().backward()
    assert (x.grad.abs() < 1e-4).all()                   # a layer norm's sum does not depend on x: 40 values of half a step


def test_streams_and_graph():
    """Another stream than the tensors' own, and a captured forward + backward replayed on new values, each replay compared
    with the eager call."""
    x, dy = make(64, 700, torch.float16).cuda(), make(64, 700, torch.float16, seed=1).cuda()
    gamma = torch.linspace(0.5, 1.5, 700, device='cuda')
    want = K.layer_norm_fwd(x, gamma)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.layer_norm_fwd(x, gamma)
    with K.launch_on(side):
        again = K.layer_norm_fwd(x, gamma)
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, again):
        assert torch.equal(a, b) and torch.equal(a, c)

    dg, db = torch.zeros(700, device='cuda'), torch.zeros(700, device='cuda')
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean, rstd = K.layer_norm_fwd(x, gamma)
        dx = K.layer_norm_bwd(dy, x, mean, rstd, gamma, dg, db)
    for seed in range(4):
        x.copy_(make(64, 700, torch.float16, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        y2, m2, r2 = K.layer_norm_fwd(x, gamma)
        dg2, db2 = torch.empty_like(dg), torch.empty_like(db)
        dx2 = K.layer_norm_bwd(dy, x, m2, r2, gamma, dg2, db2)
        for a, b in ((y, y2), (dx, dx2), (dg, dg2), (db, db2)):
            assert torch.equal(a, b)


def test_rows_far_apart_and_results_beyond_32_bits():
    """Rows 2^30 values apart (offsets pass 2^31), and more than 2^31 values in all: a row does not depend on the others."""
    ld = 2 ** 30 + 64
    far = torch.empty(3 * ld, device='cuda', dtype=torch.bfloat16)
    x, dy = (far.as_strided((3, 1000), (ld, 1), at) for at in (0, 2000))
    x.copy_(make(3, 1000, torch.bfloat16))
    dy.copy_(make(3, 1000, torch.bfloat16, seed=1))
    for a, b in zip(K.layer_norm_fwd(x), K.layer_norm_fwd(x.contiguous())):
        assert torch.equal(a, b)
    _, mean, rstd = K.layer_norm_fwd(x)
    assert torch.equal(K.layer_norm_bwd(dy, x, mean, rstd, addend=dy), K.layer_norm_bwd(dy.contiguous(), x.contiguous(), mean, rstd, addend=dy))
    del far, x, dy
    x = torch.empty((2 ** 19 + 3, 4096), device='cuda', dtype=torch.bfloat16).normal_()
    y, mean, rstd = K.layer_norm_fwd(x)
    for a, b in zip((y, mean, rstd), K.layer_norm_fwd(x[-5:])):
        assert torch.equal(a[-5:], b)
    dx = K.layer_norm_bwd(y, x, mean, rstd)
    assert torch.equal(dx[-5:], K.layer_norm_bwd(y[-5:], x[-5:], mean[-5:], rstd[-5:]))


def test_parameters_of_very_long_rows():
    """More columns than one launch has threads for: two rows, so a column's sum is one addition of fp32 products (three roundings
    each, of x - mean, times rstd, times dy)."""
    D = 2 ** 27 + 5
    x, dy = torch.empty((2, D), device='cuda').normal_(), torch.empty((2, D), device='cuda').normal_()
    mean, rstd = torch.tensor([0.25, -0.5], device='cuda'), torch.tensor([1.5, 0.75], device='cuda')
    dg, db = torch.empty(D, device='cuda'), torch.empty(D, device='cuda')
    assert K.layer_norm_bwd(dy, x, mean, rstd, None, dg, db, need_dx=False) is None
    for lo in range(0, D, 2 ** 25):
        X, Y = x[:, lo:lo + 2 ** 25].double(), dy[:, lo:lo + 2 ** 25].double()
        each = Y * (X - mean.double()[:, None]) * rstd.double()[:, None]
        assert ((dg[lo:lo + 2 ** 25].double() - each.sum(0)).abs() <= 5 * U * each.abs().sum(0) + 1e-37).all()
        assert ((db[lo:lo + 2 ** 25].double() - Y.sum(0)).abs() <= U * Y.sum(0).abs() + 1e-37).all()


def test_two_graphs_in_turn():
    """Two captured backward passes with partial sums of their own, replayed one behind the other with eager calls between."""
    sets, graphs, outs = [], [], []
    for seed, D in ((0, 700), (1, 5000)):
        x, dy = make(90, D, torch.float32, seed=seed).cuda(), make(90, D, torch.float32, seed=seed + 5).cuda()
        y, mean, rstd = K.layer_norm_fwd(x)
        sets.append((dy, x, mean, rstd, None, torch.empty(D, device='cuda'), torch.empty(D, device='cuda')))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(K.layer_norm_bwd(*sets[-1]))
        graphs.append(graph)
    for _ in range(3):
        for s in sets:
            s[0].mul_(-0.5)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for s, dx in zip(sets, outs):
            dg, db = torch.empty_like(s[5]), torch.empty_like(s[6])
            assert torch.equal(dx, K.layer_norm_bwd(*s[:5], dg, db))
            assert torch.equal(s[5], dg) and torch.equal(s[6], db)
