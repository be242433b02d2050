"""Group normalisation before a relu: what passes at the ends of fp32's range."""

import pytest
import torch

pytestmark = pytest.mark.gpu

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
