"""Newton-Schulz products of mixed lists (kernels.orthogonalize, kernels.muon_step): a matrix is as exact beside others as alone.

Tolerance: the error against float64 is that of the steps in X in float32, within a factor of two, in the mean over eight matrices.
u = 2^-24, a rounding's root mean square is 0.58 u: a product in float32 is off by its sum's and its result's, 0.82 u |L| |R| together;
with operands as two f16 pieces by those, by both operands' and by the product of the second pieces that is left out: 1.2 u, 1.5
times as much, and what follows a product is the same on both sides.  Eight matrices of 16 directions and more: each side's mean is
known to 1 / sqrt(128) = 9 %, their quotient to 12 %, two of those make 1.5 a 1.9."""
import pytest
import torch

from luminoth_amd import kernels as K

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)
# short sides beside long matrices, squares beside long ones, the shapes of a detector's heads and last blocks
LISTS = [[(16, 16), (40, 40), (100, 220), (512, 2048)],
         [(16, 20), (20, 16), (300, 300), (512, 512), (300, 5000)],
         [(512, 48), (512, 24), (1024, 81), (256, 128), (512, 128), (1152, 128), (512, 256), (1024, 320), (2304, 512)],
         [(64, 64), (128, 300), (17, 1000), (800, 65)],
         [(130, 130), (160, 200), (1500, 150)]]


def ns(u, dtype, steps=5):
    x = u.to(dtype)
    x = x / torch.linalg.norm(x)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    for _ in range(steps):
        g = x @ x.t()
        x = COEF[0] * x + (COEF[1] * g + COEF[2] * (g @ g)) @ x
    return x.t() if tall else x


@pytest.mark.parametrize('shapes', LISTS)
def test_a_matrix_is_as_exact_beside_others(shapes):
    plain, own = [0.0] * len(shapes), [0.0] * len(shapes)
    for seed in range(8):
        g = torch.Generator().manual_seed(seed)
        mats = [torch.randn(s, generator=g).cuda() for s in shapes]
        for i, (u, o) in enumerate(zip(mats, K.orthogonalize(mats))):
            want = ns(u, torch.float64)
            size = float(torch.linalg.norm(want))
            plain[i] += float(torch.linalg.norm(ns(u, torch.float32).double() - want)) / size
            own[i] += float(torch.linalg.norm(o.double() - want)) / size
    assert all(o <= 2 * p for o, p in zip(own, plain)), list(zip(shapes, own, plain))


@pytest.mark.parametrize('steps', [1, 2, 3, 4, 5, 6, 7])
def test_steps_of_matrices_that_go_different_ways(steps):
    """Short sides step by step, sides of 128 and of 256 with two and three steps in A, in one list: every matrix has taken exactly
    `steps` steps.  The bound of one step grows by the quintic's largest slope 3.4445 a step: an error of 2^-22 (1 + sqrt(k) / 64) a
    product, 3.4445^steps of it in all and one more for each step."""
    shapes = [(20, 30), (30, 200), (140, 300), (400, 130), (260, 600), (700, 300), (300, 310)]
    g = torch.Generator().manual_seed(steps)
    mats = [torch.randn(s, generator=g).cuda() for s in shapes]
    for u, o in zip(mats, K.orthogonalize(mats, steps=steps)):
        want = ns(u, torch.float64, steps)
        d = 2.0 ** -22 * (1 + max(u.shape) ** 0.5 / 64)
        err = float(torch.linalg.norm(o.double() - want))
        assert err <= (steps + 1) * 3.4445 ** steps * d + 2.0 ** -24 * float(torch.linalg.norm(want)), (tuple(u.shape), err)


def test_the_update_of_a_small_weight_beside_large_ones():
    """The optimizer's step: w - w0 = -O(g) for rate and scale 1, without momentum."""
    shapes = [(16, 20), (40, 40), (512, 1100)]
    plain, own = [0.0] * 3, [0.0] * 3
    for seed in range(8):
        g = torch.Generator().manual_seed(seed)
        grads = [torch.randn(s, generator=g).cuda() for s in shapes]
        w = [torch.zeros_like(t) for t in grads]
        K.muon_step(w, grads, [torch.zeros_like(t) for t in grads], lr=1.0, momentum=0.0, nesterov=False, scale=[1.0] * 3)
        for i, (u, o) in enumerate(zip(grads, w)):
            want = ns(u, torch.float64)
            size = float(torch.linalg.norm(want))
            plain[i] += float(torch.linalg.norm(ns(u, torch.float32).double() - want)) / size
            own[i] += float(torch.linalg.norm(-o.double() - want)) / size
    assert all(o <= 2 * p for o, p in zip(own, plain)), list(zip(shapes, own, plain))


@pytest.mark.parametrize('rows,cols', [(64, 256), (128, 500), (1000, 300), (512, 512)])
def test_rows_of_very_different_size(rows, cols):
    """Rows (the short side's) graded from 1 to 1e-6 of the largest: every row's own error.  X is held as two f16 pieces with a scale of 2^15, so
    below some size its entries are multiples of 2^-24 / 2^15 = 2^-39: a root mean square of 2^-39 / sqrt(12) an entry, sqrt(n) times that a row,
    in the first X and in that of every step, each grown 3.4445 times a step from there on: 3.4445^5 (1 + 1/11.9 + ...)^0.5 = 506 of the
    first.  What the polynomials' entries are off by adds some tenths of that.  Twice that, and four times what float32 is off by: the
    expected quotient is 1.5 (above), and one row's error may lie in one direction, so a mean over four seeds of half a normal
    distribution is known to 0.76 / 2 = 38 %, a quotient of two of them to 53 %, and three of those make 1.5 a 3.9."""
    m, n = min(rows, cols), max(rows, cols)
    grade = torch.logspace(0, -6, m)[:, None]
    plain, own = torch.zeros(m), torch.zeros(m)
    for seed in range(4):
        u = (torch.randn((m, n), generator=torch.Generator().manual_seed(seed)) * grade).cuda()
        want = ns(u, torch.float64)
        got = K.orthogonalize([u if rows <= cols else u.t().contiguous()])[0]
        got = got if rows <= cols else got.t()
        plain += (ns(u, torch.float32).double() - want).norm(dim=1).cpu().float() / 4
        own += (got.double() - want).norm(dim=1).cpu().float() / 4
    tol = 4 * plain + 2 * 506 * n ** 0.5 * 2.0 ** -39 / 12 ** 0.5
    assert (own <= tol).all(), float((own / tol).max())
