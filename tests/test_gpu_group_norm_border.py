"""Group normalisation before a relu: what passes forward and backward, at the ends of fp32's range and far from zero."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
# tiles held in registers (all groups in a workgroup, or some; groups of whole accesses or not), cut samples, a shape that no tile covers
SHAPES = [((64, 26, 26, 32), 8), ((40, 30, 48), 6), ((600, 26, 26, 32), 8), ((9, 40, 18), 6), ((2, 30000, 32), 2), ((3, 9000, 10), 5), ((2, 3, 5000), 1)]


def _stats(x, stats, G):
    C = x.shape[-1]
    return (t.view(x.shape[0], 1, G).repeat_interleave(C // G, dim=2) for t in stats)


@pytest.mark.parametrize('size,small', [(1e10, 1e-38), (1e10, 1e-42), (1e-37, 1e-10), (1.0, 1e-44)])
@pytest.mark.parametrize('shape,G', SHAPES)
def test_products_below_the_range(dev, shape, G, size, small):
    """gamma / sqrt(var + eps), or its product with a distance, may lie below the smallest float32: the sign still decides.  With dy = 1, dbeta
    counts what passes; in 64 bits from the statistics that the operator reports."""
    from hgq2_amd import _lib

    _lib.native()
    g = torch.Generator().manual_seed(23)
    C = shape[-1]
    x = (size * torch.randn(shape, generator=g)).to(dev)
    gamma = (small * (1 + torch.rand(C, generator=g)) * torch.where(torch.arange(C) % 3 > 0, 1.0, -1.0)).to(dev)
    beta = torch.zeros(C, device=dev)
    beta[1], beta[2] = 1e-3, -1e-3
    assert (gamma != 0).all()
    y, stats = torch.ops.hgq.group_norm_fwd(x, gamma, beta, G, 1e-3, 1)
    mean, rstd = _stats(x, stats, G)
    passes = (x.view(shape[0], -1, C).double() - mean) * (rstd * gamma.double()) + beta.double() > 0
    _, _, dbeta = torch.ops.hgq.group_norm_bwd(torch.ones_like(x), x, gamma, beta, stats, G, 1, True, True, True)
    assert torch.equal(dbeta.double(), passes.sum(dim=(0, 1)).double())  # (counts below 2^24 are exact)


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16])
@pytest.mark.parametrize('shape,G', SHAPES)
def test_one_border_for_both_passes(dev, shape, G, dtype):
    """A mean of 3000 standard deviations (fp16: of 50, more of it than its spacing allows there would be no data): its rounding to fp32 is 1e-4
    of them, and must not decide whether y is zero.

    z from x - mean, in units of u = 2^-24: the difference u, the scale (statistic and product) 2 u, z itself u, all of |xhat gamma| at
    most; beta with the mean's rest u of itself, and that rest, at most 2^-24 of the mean, 3 u of itself: nothing.  Beyond 5 u (|xhat
    gamma| + |beta|), y > 0 and what passes backward have to agree (fp16: where z is not rounded to zero)."""
    from hgq2_amd import _lib

    _lib.native()
    g = torch.Generator().manual_seed(24)
    C = shape[-1]
    x = (torch.randn(shape, generator=g) + (3000.0 if dtype == torch.float32 else 50.0)).to(dtype).to(dev)
    gamma = ((1 + 0.3 * torch.randn(C, generator=g)) * torch.where(torch.arange(C) % 3 > 0, 1.0, -1.0)).to(dev)
    beta = (0.5 * torch.randn(C, generator=g)).to(dev)
    # every channel's beta puts its border on an element of the first sample, to within fp32's rounding of beta
    _, stats = torch.ops.hgq.group_norm_fwd(x, gamma, beta, G, 0.0, 1)
    mean, rstd = _stats(x, stats, G)
    xs = x.view(shape[0], -1, C)
    beta = (-(xs[0, 0].double() - mean[0, 0]) * rstd[0, 0] * gamma.double()).float()
    y, stats = torch.ops.hgq.group_norm_fwd(x, gamma, beta, G, 0.0, 1)
    mean, rstd = _stats(x, stats, G)
    h = (xs.double() - mean) * rstd * gamma.double()
    z = h + beta.double()
    sure = z.abs() > 5 * U * (h.abs() + beta.double().abs()) + (2.0**-24 if dtype == torch.float16 else 0.0)
    assert sure.double().mean() > 0.8  # (an element per channel lies on its border)
    assert torch.equal((y.view(xs.shape) > 0)[sure], (z > 0)[sure])
    dx, _, dbeta = torch.ops.hgq.group_norm_bwd(torch.ones_like(x), x, gamma, beta, stats, G, 1, True, True, True)
    assert torch.equal(dbeta.double(), (z > 0).sum(dim=(0, 1)).double())


@pytest.mark.parametrize('shape,G', SHAPES)
def test_a_mean_far_from_zero_before_a_relu(dev, shape, G):
    """y itself under the same data: 3 u of xhat and u of the rest are all that the mean's place leaves (the variance: 2 L u of the definition's
    bound for sums of at most 64 terms in a row and 32 levels, L = 96, in 64 bits here, so u)."""
    from hgq2_amd import ops

    g = torch.Generator().manual_seed(25)
    C = shape[-1]
    x = (torch.randn(shape, generator=g) + 3000.0).to(dev)
    gamma, beta = (1 + 0.3 * torch.randn(C, generator=g)).to(dev), (0.5 * torch.randn(C, generator=g)).to(dev)
    y = ops.group_norm(x, G, gamma, beta, 0.0, 'relu').view(shape[0], -1, C)
    t = x.double().view(shape[0], -1, G, C // G)
    mean = t.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / ((t - mean) ** 2).mean(dim=(1, 3), keepdim=True).sqrt()
    h = ((t - mean) * rstd).reshape(y.shape) * gamma.double()
    want = (h + beta.double()).clamp(min=0)
    # (the statistics in 64 bits are those of x about its fp32 mean: off by the square of 2^-13, relatively half of that squared deviation)
    tol = 6 * U * (h.abs() + beta.double().abs()) + h.abs() * 2.0**-26
    worst = float(((y.double() - want).abs() / tol).max())
    assert worst <= 1, worst
