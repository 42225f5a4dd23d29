"""Alternatives of rows with not-a-number (kernels.log_probs_fwd): those classes come first, in the order of their index, then the
others by value - at class 0 and in rows of nothing else too, whatever way a row is cut up."""
import math

import pytest
import torch

from luminoth_amd import kernels as K

pytestmark = pytest.mark.gpu


def order(x, k):
    """float64 on the CPU: not-a-number first, larger values, lower indices"""
    x = torch.where(torch.isnan(x), torch.full_like(x, math.inf), x)
    return torch.sort(x + 0.0, dim=-1, descending=True, stable=True).indices[:, :k]


# (rows, classes): a wave, a block of 256 and of 1024 threads a row, parts of a row, several segments a part
CUTS = [(3, 4), (5, 64), (7, 81), (4, 1024), (9, 5000), (300, 3000), (3, 70001), (2, 300007), (2100, 16389)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('rows,C', CUTS)
def test_not_a_number(rows, C, dtype):
    g = torch.Generator(device='cuda').manual_seed(rows + C)
    x = (torch.randn((rows, C), generator=g, device='cuda') * 3).to(dtype)
    x[0, 0] = math.nan
    x[1] = math.nan
    if rows > 2:
        x[2, 0] = x[2, C - 1] = x[2, C // 2] = math.nan
        x[2, 1] = -math.inf
    if rows > 3:
        x[3, C // 2:] = math.nan
        x[3, 0] = math.nan
    for k in sorted({1, 2, 20, 64, C}):
        if k > min(64, C):
            continue
        logp, entropy, top, index, lse = K.log_probs_fwd(x, torch.zeros(rows, dtype=torch.int64, device='cuda'), k)
        n = min(rows, 4)
        assert torch.equal(index[:n].cpu(), order(x[:n].cpu().double(), k)), k
        assert torch.isnan(top[:n]).all() and torch.isnan(logp[:n]).all() and torch.isnan(entropy[:n]).all() and torch.isnan(lse[:n]).all()
        assert (index >= 0).all() and (index < C).all()


@pytest.mark.parametrize('C', [4, 21, 64])
def test_every_class_is_an_alternative(C):
    """top = all classes of a diverged head: every index once, and the gradient of such a row is not a number everywhere"""
    x = torch.full((6, C), math.nan, device='cuda')
    x[1, 1:] = 0.5
    x[2, :-1] = 0.5
    x[3] = -math.inf
    x[3, 0] = math.nan
    x[4] = math.inf
    x[5] = -math.inf
    _, entropy, top, index, lse = K.log_probs_fwd(x, None, C)
    assert torch.equal(index.cpu().sort(-1).values, torch.arange(C).expand(6, C))
    assert torch.equal(index.cpu()[:4], order(x[:4].cpu().double(), C))
    assert torch.equal(index[4:].cpu(), torch.arange(C).expand(2, C))
    dx = K.log_probs_bwd(x, None, lse, entropy, None, torch.ones(6, device='cuda'), index, torch.ones((6, C), device='cuda'))
    assert torch.isnan(dx[:5]).all() and (dx[5] == 0).all()


def test_alternatives_of_a_diverged_head():
    """What model.rcnn.top_alternatives hands out for (images, proposals, classes) of nothing but not-a-number"""
    x = torch.full((2, 300, 21), math.nan, device='cuda')
    index = K.log_probs_fwd(x, None, 21)[3]
    assert torch.equal(index.cpu(), torch.arange(21).expand(2, 300, 21))


@pytest.mark.parametrize('rows,C,dtype', [(2100, 16389, torch.float32), (1400, 33001, torch.bfloat16), (4200, 16390, torch.float16), (3, 300007, torch.float32)])
@pytest.mark.parametrize('k', [20, 33, 40, 64])
def test_sums_with_and_without_alternatives(rows, C, dtype, k):
    """More alternatives cut long rows into other parts, so sums are added in another order: log p, lse and entropy of both ways are each
    within (100 + 4 E|z|) u of the exact ones (entropy: 110 E|z| + 4 E z^2 more; their own rounding on top), u = 2^-24, z = x - max."""
    g = torch.Generator(device='cuda').manual_seed(C + k)
    x = (torch.randn((rows, C), generator=g, device='cuda') * 3).to(dtype)
    x[0] = torch.linspace(-9, 9, C, device='cuda')
    x[1] = 1.5
    x[2, : C - 5] = -math.inf
    t = torch.randint(C - 5, C, (rows,), generator=g, device='cuda')
    n = min(rows, 300)
    a, b = ([v[:n].double() for v in (r[0], r[4], r[1])] for r in (K.log_probs_fwd(x, t, k), K.log_probs_fwd(x, t, 0)))
    z = x[:n].double()
    z = z - z.amax(-1, keepdim=True)
    p = torch.softmax(z, -1)
    z = torch.where(p > 0, z, torch.zeros_like(z))
    ez, ezz = (p * z.abs()).sum(-1), (p * z * z).sum(-1)
    u = 2.0 ** -24
    for v, w, more in zip(a, b, (0, 0, 110 * ez + 4 * ezz)):
        assert ((v - w).abs() <= 2 * u * (100 + 4 * ez + more) + 4 * u * w.abs()).all()
