"""Group normalisation, backward: sums of very many equal terms.

Equal terms added one after the other in fp32 are rounded the same way within a binade, so n of them drift by up to n / 2 units of u = 2^-24,
which random terms never show.  The bounds are those of the 64-bit comparison: no sum adds more than 64 terms in a row before it goes on
pairwise in at most 32 levels, L = 96 of u; dgamma and dbeta twice that, within a sample and over the samples."""

import pytest
import torch

from .test_gpu_group_norm import _check, _definition

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('B,C', [(100_003, 1025), (40_009, 2050)])
def test_many_samples_without_a_tile(dev, B, C, dtype):
    """Rows that no tile covers, one position per sample: each sample leaves its terms of dgamma and dbeta, the sums over all are what
    counts.  dy has one value per channel."""
    from hgq2_amd import ops

    g = torch.Generator(device=dev).manual_seed(28)
    x = torch.randn(B, 1, C, generator=g, device=dev).to(dtype)
    dy = (torch.rand(C, generator=g, device=dev) + 0.5).to(dtype)
    gamma, beta = torch.ones(C, device=dev, requires_grad=True), torch.zeros(C, device=dev, requires_grad=True)
    y = ops.group_norm(x, 1, gamma, beta)
    dgamma, dbeta = torch.autograd.grad(y, [gamma, beta], dy.expand(B, 1, C))
    del y
    sums, tols = [0, 0], [0, 0]
    for at in range(0, B, 5000):
        part = x[at:at + 5000]
        want, tol = _definition(part, dy.expand(len(part), 1, C), gamma.detach(), beta.detach(), 1, 1e-3, 'linear')
        for k in range(2):
            sums[k], tols[k] = sums[k] + want[2 + k], tols[k] + tol[2 + k]
    _check(dbeta, sums[1], tols[1], torch.float32, 'dbeta')
    _check(dgamma, sums[0], tols[0], torch.float32, 'dgamma')


@pytest.mark.parametrize('C,G,dtype', [(32, 32, torch.float32), (32, 8, torch.float32), (32, 32, torch.bfloat16)])
def test_one_long_sample(dev, C, G, dtype):
    """A sample cut into thousands of runs, with dy = 1 and one gamma per group: d is its own mean, dx zero but for the rounding of the two means."""
    from hgq2_amd import ops

    S = (1 << 21) + 77
    g = torch.Generator(device=dev).manual_seed(29)
    x = torch.randn(1, S, C, generator=g, device=dev).to(dtype).requires_grad_(True)
    gamma = (torch.rand(G, generator=g, device=dev) + 0.5).repeat_interleave(C // G)
    y = ops.group_norm(x, G, gamma)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    want, tol = _definition(x.detach(), torch.ones_like(y), gamma, None, G, 1e-3, 'linear')
    _check(dx, want[1], tol[1], dtype, 'dx')
