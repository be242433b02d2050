"""Norms around a residual sum: sums do not lose more as rows, or channels beyond what a workgroup holds, become many.

u = 2^-24.  Rows of ones have norms of one (relatively off by 4 u: the mean, the root, the product), so with an upstream gradient c in every place dpost and dpre are
rows * c and a sample's dgate its rows * c.  A thread adds at most 64 rows one after the other, 64 bits join teams of a workgroup (256 threads over the
row's threads) and the rest: 64 u (and one for each team, which they were once allowed); a gate's sums meet once more over a slice's units, at most 64 in all with the rows: 2 u, and the factors 8 u.  c has the property that adding
it up 512 times in fp32 is off by 128 u, a bias that grows with every further row."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
C0 = float.fromhex('0x1.03b9p+0')


# rows of a wavefront and of several, whose sums lie in registers, in LDS and in memory; workgroups with one unit each, units of a sample, samples of many units
@pytest.mark.parametrize('batch,positions,channels,gate', [(1, 1 << 20, 512, None), (1, 3 << 19, 512, 'element'), (2, 3 << 18, 512, 'sample'), (800, 2048, 512, 'sample'), (70000, 3, 512, 'sample'),
                                                           (1, 1 << 18, 2048, None), (800, 512, 2048, 'sample'), (1, 1 << 17, 8192, None), (1, 1 << 17, 8208, None), (300, 512, 8208, 'sample')])
def test_sums_over_many_rows(dev, batch, positions, channels, gate):
    from hgq2_amd import ops

    shape, rows = (batch, positions, channels), batch * positions
    tol = (64 + max(1, 256 // max(1, channels // 8)) + 14) * U
    x = torch.ones(shape, device=dev)
    c = torch.full(shape, C0, device=dev)
    post, pre = (torch.ones(channels, device=dev, requires_grad=True) for _ in range(2))
    g = None if gate is None else torch.ones(shape if gate == 'element' else (batch, channels), device=dev, requires_grad=gate == 'sample')
    y, h = ops.residual_norm(x, x, post, pre, g, None, epsilon=0.0)
    want = rows * C0
    leaves = [post] + ([g] if gate == 'sample' else [])
    grads = torch.autograd.grad(y, leaves, c, retain_graph=True)
    assert float((grads[0].double() - want).abs().max()) <= tol * want, float((grads[0].double() / want - 1).abs().max()) / U
    if gate == 'sample':
        assert float((grads[1].double() / (positions * C0) - 1).abs().max()) <= tol
    (got,) = torch.autograd.grad(h, [pre], c)
    assert float((got.double() - want).abs().max()) <= tol * want, float((got.double() / want - 1).abs().max()) / U


@pytest.mark.parametrize('rows,channels,gate', [(1 << 17, 8, None), (1 << 17, 8, 'sample'), (1 << 17, 3, None), (1 << 16, 16, 'element')])
def test_sums_of_many_teams(dev, rows, channels, gate):
    """A row or two a thread, 128 or 256 teams a workgroup, which meet in 64 bits: 2 + 14 u.  Adding this c up 256 times in fp32 is off by 64 u."""
    from hgq2_amd import ops

    c0 = float.fromhex('0x1.ff73p+0')
    shape = (2, rows // 2, channels)
    x, c, post = torch.ones(shape, device=dev), torch.full(shape, c0, device=dev), torch.ones(channels, device=dev, requires_grad=True)
    g = None if gate is None else torch.ones(shape if gate == 'element' else (2, channels), device=dev, requires_grad=gate == 'sample')
    y, _ = ops.residual_norm(x, x, post, None, g, None, epsilon=0.0)
    grads = torch.autograd.grad(y, [post] + ([g] if gate == 'sample' else []), c)
    assert float((grads[0].double() / (rows * c0) - 1).abs().max()) <= 16 * U
    if gate == 'sample':
        assert float((grads[1].double() / (rows // 2 * c0) - 1).abs().max()) <= 16 * U


@pytest.mark.parametrize('rows,channels,P,gate', [(70, 8208, 1, None), (700, 40, 1, None), (66000, 8, 2, 'sample'), (40000, 333, 400, 'sample'), (3000, 1000, 3, 'sample')])
def test_slices_of_every_workgroup_are_written(dev, rows, channels, P, gate):
    """Random rows, as many that some workgroups leave a slice more than others; the same sums in 64 bits.  Relatively to the sum of magnitudes: as above, and 80 u for the terms, whose
    norms go through sums of a row."""
    from hgq2_amd import ops

    g = torch.Generator(device=dev).manual_seed(rows)
    x, u, dy, dh = (torch.randn(rows // P, P, channels, generator=g, device=dev) for _ in range(4))
    post, pre = (torch.rand(channels, generator=g, device=dev) + 0.5 for _ in range(2))
    gt = torch.randn(rows // P, channels, generator=g, device=dev) if gate else None
    leaves = [t.clone().requires_grad_(True) for t in (post, pre)]
    got = torch.autograd.grad(ops.residual_norm(x, u, leaves[0], leaves[1], gt), leaves, [dy, dh])
    x, u, dy, dh, post, pre = (t.double() for t in (x, u, dy, dh, post, pre))
    open_ = gt.double()[:, None] if gate else torch.ones((), dtype=torch.float64, device=dev)
    n = u / torch.sqrt((u * u).mean(-1, keepdim=True) + 1e-6)
    y = x + n * post * open_
    r = 1 / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6)
    m, e = y * r, dh * pre
    s = (e * m).mean(-1, keepdim=True)
    dx = dy + r * (e - m * s)
    size = dy.abs() + r * (e.abs() + m.abs() * (e * m).abs().mean(-1, keepdim=True))  # (dx's roundings are relative to what it is formed of)
    teams = max(1, 256 // max(1, channels // 8))
    for a, b, magnitude in ((got[0], dx * open_ * n, size * (open_ * n).abs()), (got[1], dh * m, (dh * m).abs())):
        tol = (64 + teams + 94) * U * magnitude.sum((0, 1))
        assert ((a.double() - b.sum((0, 1))).abs() <= tol).all()


@pytest.mark.parametrize('channels', [(1 << 24) + 5, 300_000])
def test_means_of_very_many_channels(dev, channels):
    """Rows of one value have a norm of one.  A thread adds four products in fp32 and such sums in 64 bits, 1024 threads meet pairwise: 4 + 10 u, with the factors' roundings 20 u; a
    gradient of one value leaves e - m mean(e m) = 0, off by twice that of e."""
    from hgq2_amd import ops

    v = 1.1
    x = torch.full((2, channels), v, device=dev, requires_grad=True)
    u = torch.full((2, channels), v, device=dev, requires_grad=True)
    h = ops.rms_norm(x, epsilon=0.0)
    assert float((h.double() - 1).abs().max()) <= 20 * U
    dh = torch.full_like(x, C0)
    (dx,) = torch.autograd.grad(h, [x], dh)
    assert float(dx.abs().max()) <= 2 * 20 * U * C0 / v
    y, h = ops.residual_norm(x, u, epsilon=0.0)
    assert float((y.double() - (float(x[0, 0]) + 1)).abs().max()) <= 24 * U * (v + 1)
    dx, du = torch.autograd.grad([y, h], [x, u], [dh, dh])
    assert float((dx.double() - C0).abs().max()) <= 2 * 24 * U * C0 and float(du.abs().max()) <= 2 * 40 * U * C0 / v


def test_gradients_of_more_gammas_than_a_launch_has_threads_for(dev):
    """Two rows of ones and twos have norms of one: dgamma is the sum of two upstream gradients, exact."""
    from hgq2_amd import ops

    channels = (1 << 25) + 37
    x = torch.tensor([[1.0], [2.0]], device=dev).expand(2, channels).contiguous()
    gamma = torch.ones(channels, device=dev, requires_grad=True)
    dh = torch.randint(-8, 9, (2, channels), device=dev).float()
    (dg,) = torch.autograd.grad(ops.rms_norm(x, gamma, epsilon=0.0), [gamma], dh)
    assert float((dg.double() - dh.double().sum(0)).abs().max()) <= 40 * U * 16  # (the norms' own: 20 u each)
