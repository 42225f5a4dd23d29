"""Newton-Schulz products (kernels.orthogonalize) and the optimizer step on them (kernels.muon_step, train.optimizer.type: muon)
against the formulas in float64.

Tolerance of O(U).  A product of m x k by k x n numbers with operands of error 2^-24 and fp32 accumulation is off, in the 2-norm
of its entries, by at most d |L|_F |R|_2 with d = 2^-22 (1 + sqrt(k) / 64) (operands 2 * 2^-24, three partial products, k / 16
rounded additions that add up like a random walk).  What is off by e in X is off by 3.4445 e at most one step later (the
quintic's largest slope, at 0), and |X_k|_F <= min(3.4445^k, 1.25 sqrt(m)).  Five steps: at most (5 + 1) 3.4445^5 d = 2910 d in
all, and the result is rounded once to its type."""
import math

import pytest
import torch

from luminoth_amd import kernels as K

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)
SHAPES = [(1, 1), (1, 9), (7, 1), (3, 5), (16, 16), (64, 64), (65, 63), (33, 200), (200, 33), (128, 128), (129, 257), (130, 100),
          (300, 1000), (1024, 320), (72, 2304), (2304, 64), (512, 512)]


def ns(u, steps=5, eps=1e-7):
    u = u.double()
    x = u / max(float(torch.linalg.norm(u)), eps)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    for _ in range(steps):
        g = x @ x.t()
        x = COEF[0] * x + (COEF[1] * g + COEF[2] * (g @ g)) @ x
    return x.t() if tall else x


def bound(u, steps=5):
    d = 2.0 ** -22 * (1 + math.sqrt(max(u.shape)) / 64)
    return (steps + 1) * 3.4445 ** steps * d


def close(got, u, steps=5, eps=1e-7):
    want = ns(u, steps, eps)
    err = float(torch.linalg.norm(got.cpu().double() - want))
    half = torch.finfo(got.dtype).eps / 2
    assert err <= bound(u, steps) + half * float(torch.linalg.norm(want)) + (2.0 ** -25 * want.numel() ** 0.5 if got.dtype == torch.float16 else 0), \
        (tuple(u.shape), err, bound(u, steps))


def make(rows, cols, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + rows * 101 + cols)
    r = min(4, rows, cols)
    return scale * (0.3 * torch.randn((rows, r), generator=g) @ torch.randn((r, cols), generator=g) + torch.randn((rows, cols), generator=g))


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('rows,cols', SHAPES)
def test_orthogonalize(rows, cols, dtype):
    u = make(rows, cols).to(dtype)
    out, = K.orthogonalize([u.cuda()])
    assert out.dtype == dtype and out.shape == u.shape
    close(out, u)


def test_many_matrices_at_once():
    """More shapes and matrices than one launch takes; HWIO kernels count as (inputs, out); a matrix alone."""
    mats = [make(5 + 3 * (i % 31), 4 + 7 * (i % 29), seed=i) for i in range(101)] + [make(288, 40).view(3, 3, 32, 40)]
    got = K.orthogonalize([m.cuda() for m in mats])
    for m, o in zip(mats, got):
        assert o.shape == m.shape
        close(o.view(-1, o.shape[-1]), m.view(-1, m.shape[-1]))
    # how a product's k is split, and so the order of its additions, goes by the whole list: each result is within bound() of the
    # exact one, so two of them are within twice that of each other
    alone, = K.orthogonalize([mats[50].cuda()])
    close(alone, mats[50])
    assert float(torch.linalg.norm(alone.double() - got[50].double())) <= 2 * bound(mats[50])
    assert torch.equal(alone, K.orthogonalize([mats[50].cuda()])[0])
    assert K.orthogonalize([]) == []


@pytest.mark.parametrize('scale', [1e-30, 1e-3, 1e18, 1e37])
def test_scales(scale):
    """|U|^2 leaves float32's range; below eps the quotient is U / eps, as defined."""
    u = make(40, 90, scale=scale)
    out, = K.orthogonalize([u.cuda()])
    close(out, u)


def test_zero_steps_eps_and_not_a_number():
    z = torch.zeros((70, 30), device='cuda')
    assert (K.orthogonalize([z])[0] == 0).all()
    bad = make(70, 30)
    bad[3, 4] = math.nan
    good = make(70, 30)
    a, b = K.orthogonalize([bad.cuda(), good.cuda()])
    assert torch.isnan(a).all()
    close(b, good)
    for steps in (1, 2, 3, 8):
        close(K.orthogonalize([good.cuda()], steps=steps)[0], good, steps=steps)
    close(K.orthogonalize([good.cuda()], eps=1e3)[0], good, eps=1e3)


@pytest.mark.parametrize('nesterov', [True, False])
def test_step(nesterov):
    """Two steps with everything on: weight decay, gradient factors and scale, a rate per matrix; tensors are views of one buffer."""
    shapes = [(96, 64), (3, 3, 16, 40), (200, 300), (64, 64), (5, 2)]
    n = [math.prod(s) for s in shapes]
    g = torch.Generator().manual_seed(3)
    w, v, gr = (torch.randn(sum(n) + 8, generator=g) for _ in range(3))

    def views(flat):
        out, at = [], 4
        for s, k in zip(shapes, n):
            out.append(flat[at:at + k].view(s))
            at += k
        return out
    dw, dv, dg = w.cuda(), v.cuda(), gr.cuda()
    wd, scale = [0.0, 0.1, 0.01, 0.0, 0.3], [1.0, 0.5, 2.0, 0.1, 1.0]
    factors = torch.tensor([1.0, 0.5, 0.25, 1.0, 0.125])
    rw, rv, rg = ([t.double() for t in views(f)] for f in (w, v, gr))
    tol = [0.0] * 5
    for _ in range(2):
        K.muon_step(views(dw), views(dg), views(dv), lr=0.3, momentum=0.9, nesterov=nesterov, weight_decay=wd, scale=scale,
                    factors=factors.cuda(), gscale=0.5)
        for i in range(5):
            gp = (0.5 * rg[i] + wd[i] * rw[i]) * float(factors[i])
            rv[i] = 0.9 * rv[i] + gp
            u = (gp + 0.9 * rv[i] if nesterov else rv[i]).reshape(-1, shapes[i][-1])
            # the update's input is off by some roundings of its terms too: 4 * 2^-24 of its norm, times the slope
            tol[i] += 0.3 * scale[i] * 2 * bound(u)
            rw[i] = rw[i] - 0.3 * scale[i] * ns(u).reshape(shapes[i])
    for i in range(5):
        a, b = views(dw)[i].cpu().double(), views(dv)[i].cpu().double()
        assert float(torch.linalg.norm(a - rw[i])) <= tol[i] + 2.0 ** -22 * float(torch.linalg.norm(rw[i]))
        assert float(torch.linalg.norm(b - rv[i])) <= 2.0 ** -21 * float(torch.linalg.norm(rv[i])) + wd[i] * tol[i]
    assert torch.equal(dg.cpu(), gr)
    for flat, start in ((dw, w), (dv, v)):                 # what lies around the matrices
        assert torch.equal(flat[:4].cpu(), start[:4]) and torch.equal(flat[-4:].cpu(), start[-4:])


def test_same_bits_streams_and_graph():
    mats = [make(300, 200).cuda(), make(64, 640).cuda(), make(20, 10).cuda()]
    want = K.orthogonalize(mats)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.orthogonalize(mats)
    with K.launch_on(side):
        again = K.orthogonalize(mats)
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, again):
        assert torch.equal(a, b) and torch.equal(a, c)
    # two captured graphs and eager calls in turn: no scratch memory is shared
    other = [make(300, 200, seed=5).cuda(), make(64, 640, seed=6).cuda()]
    graphs, outs = [], []
    for inputs in (mats, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(K.orthogonalize(inputs))
        graphs.append(graph)
    for seed in range(3):
        mats[0].copy_(make(300, 200, seed=seed))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for inputs, got in ((mats, outs[0]), (other, outs[1])):
            for a, b in zip(got, K.orthogonalize(inputs)):
                assert torch.equal(a, b)


@pytest.mark.parametrize('rows,cols', [(1000, 2100), (1500, 1600), (5000, 1400), (4100, 4200), (4000, 9000), (2900, 8800), (8800, 2900)])
def test_large_matrices(rows, cols):
    """More tiles than one round of blocks takes: the last ones are split along k and joined; products with X in tiles of 256 rows,
    of which the last has 128; the reference on the device too."""
    u = make(rows, cols).cuda()
    out, = K.orthogonalize([u])
    want = ns(u)
    assert float(torch.linalg.norm(out.double() - want)) <= bound(u) + 2.0 ** -24 * float(torch.linalg.norm(want))


def test_norms_at_the_ends_of_the_range():
    """8192 / |U|_F, the factor of the planes, beyond fp32's range at both ends (and below its normal numbers)."""
    tiny = make(40, 90, scale=1e-36)
    close(K.orthogonalize([tiny.cuda()], eps=1e-38)[0], tiny, eps=1e-38)
    huge = make(2600, 2700).clamp(-3.0, 3.0) * 1e38
    out, = K.orthogonalize([huge.cuda()])
    want = ns(huge.cuda())
    assert float(torch.linalg.norm(out.double() - want)) <= bound(huge) + 2.0 ** -24 * float(torch.linalg.norm(want))


def test_many_steps_stay_in_the_band():
    """The quintic takes [0.68, 1.21] into itself (its extremes there: 1.2025 at 0.5545 from below, 0.682 at 1.0501), and every
    singular value that fp32 can tell from zero gets there in 64 steps; rounding adds 2^-20 at most a step, which the slopes
    in the band (below 3.5 in magnitude) do not let grow past 2^-17 while a value moves to and fro inside it."""
    u = make(64, 96)
    s = torch.linalg.svdvals(K.orthogonalize([u.cuda()], steps=64)[0].cpu().double())
    assert s.min() >= 0.67 and s.max() <= 1.22


def test_one_gradient_for_two_weights():
    w = [make(48, 32, seed=i).cuda() for i in range(2)]
    v = [torch.zeros_like(t) for t in w]
    g = make(48, 32, seed=7).cuda()
    w2, v2 = [t.clone() for t in w], [t.clone() for t in v]
    K.muon_step(w, [g, g], v, lr=0.1)
    K.muon_step(w2, [g.clone(), g.clone()], v2, lr=0.1)
    for a, b in zip(w + v, w2 + v2):
        assert torch.equal(a, b)


def test_matrices_that_are_not_contiguous_are_refused():
    from luminoth_amd import _lib
    u = make(48, 32).cuda()
    with pytest.raises(_lib.LuminothHipError, match='contiguous'):
        K.orthogonalize([u.t()])
    with pytest.raises(_lib.LuminothHipError, match='contiguous'):
        K.muon_step([u.t()], [u.t()], [torch.zeros_like(u).t()], lr=0.1)


@pytest.mark.parametrize('steps', [1, 2, 3, 4, 5])
def test_short_sides(steps):
    """Lists of short sides, padded ones among them: up to 64 rows, and up to 128."""
    for sizes in ([(64, 64), (40, 50), (300, 7)], [(128, 300), (33, 900), (100, 260), (800, 65)]):
        mats = [make(*s) for s in sizes]
        for m, o in zip(mats, K.orthogonalize([m.cuda() for m in mats], steps=steps)):
            close(o, m, steps=steps)


@pytest.mark.parametrize('rows,cols', [(16, 33), (20, 41), (16, 100), (40, 40), (60, 120), (100, 220), (64, 600), (127, 300), (128, 260), (200, 420),
                                       (256, 520), (320, 1024), (500, 500)])
def test_as_exact_as_fp32(rows, cols):
    """The error against float64 is that of the steps in X in fp32, within a factor of two, in the mean over eight matrices.
    u = 2^-24, a rounding's root mean square is u / sqrt(3) = 0.58 u: a product in fp32 is off by its sum's and its result's, 0.82 u
    |L| |R| together; here by those, by both operands' (their second halves end at u) and by the product of the second halves that is
    left out (u / 3): 1.2 u, 1.5 times as much, and what follows a product is the same on both sides.  Eight matrices of 16 directions
    and more: each side's mean is known to 1 / sqrt(128) = 9 %, their quotient to 12 %, two of those make 1.5 a 1.9.  Several steps in A
    without a fresh one would be off by 3 to 5 times as much where the matrix is small."""
    plain, own = 0.0, 0.0
    for seed in range(8):
        u = torch.randn((rows, cols), generator=torch.Generator().manual_seed(seed)).cuda()
        x = u / torch.linalg.norm(u)
        for _ in range(5):
            g = x @ x.t()
            x = COEF[0] * x + (COEF[1] * g + COEF[2] * (g @ g)) @ x
        want = ns(u)
        plain += float(torch.linalg.norm(x.double() - want) / torch.linalg.norm(want)) / 8
        own += float(torch.linalg.norm(K.orthogonalize([u])[0].double() - want) / torch.linalg.norm(want)) / 8
    assert own <= 2 * plain, (own, plain)


def test_one_shape_and_many():
    """A launch of one shape has a table of its own: one matrix, several of one shape, and the same ones among others."""
    a, b, c = make(90, 170), make(90, 170, seed=1), make(40, 60)
    for mats in ([a], [a, b], [a, b, c]):
        for m, o in zip(mats, K.orthogonalize([m.cuda() for m in mats])):
            close(o, m)
    w, v = [m.cuda() for m in (a, b)], [torch.zeros(90, 170, device='cuda') for _ in range(2)]
    K.muon_step(w, [m.cuda() for m in (b, a)], v, lr=1.0, momentum=0.0, nesterov=False, scale=[1.0, 1.0])
    for got, start, g in zip(w, (a, b), (b, a)):
        err = float(torch.linalg.norm(got.cpu().double() - (start.double() - ns(g))))
        assert err <= bound(g) + 2.0 ** -24 * float(torch.linalg.norm(got.cpu().double()))
