"""Group normalisation against a plain implementation in 64 bits.

Tolerances, u = 2^-24 (half a step of fp32) and L = 96: no sum of the kernels adds more than 64 terms one after the other before it goes
on pairwise, in at most 32 further levels, so a sum is off by at most L u times the sum of magnitudes.  The mean is then off by L u
mean|x| and the variance, formed about that mean, relatively by 2 L u; xhat by rstd L u mean|x| + L u |xhat|.  z adds three roundings, an
activation at most 1.1 times what z is off (the largest slope of z / (1 + exp(-z))) and 8 u of its own.  The backward formulas are carried through term by
term below (a second derivative is at most 1/2).  A 16-bit type adds half a step.  Where |z| is within its tolerance of zero the slope of
a relu may be either: such elements are left out, and counted into the sums' tolerances."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U, L = 2.0**-24, 96
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _definition(x, dy, gamma, beta, G, eps, act):
    """Values and tolerances of y, dx, dgamma, dbeta in 64 bits; x [B, S, C]."""
    x, dy = x.double(), dy.double().to(x.device)
    B, S, C = x.shape
    ga = gamma.double() if gamma is not None else torch.ones(C, dtype=torch.float64, device=x.device)
    be = beta.double() if beta is not None else torch.zeros(C, dtype=torch.float64, device=x.device)
    per = lambda t: t.view(B, S, G, C // G)  # noqa: E731
    gmean = lambda t: per(t).mean(dim=(1, 3), keepdim=True)  # noqa: E731
    whole = lambda t: t.expand(B, S, G, C // G).reshape(B, S, C)  # noqa: E731
    mean = gmean(x)
    var = ((per(x) - mean) ** 2).mean(dim=(1, 3), keepdim=True)
    rstd = whole(1 / torch.sqrt(var + eps))
    xh = (x - whole(mean)) * rstd
    t_xh = rstd * L * U * whole(gmean(x.abs())) + (L + 4) * U * xh.abs()
    z = xh * ga + be
    t_z = t_xh * ga.abs() + 3 * U * ((xh * ga).abs() + be.abs())
    p = torch.sigmoid(z)
    if act == 'relu':
        y, slope, unsure = z.clamp(min=0), (z > 0).double(), z.abs() <= t_z
    elif act == 'silu':
        y, slope, unsure = z * p, p * (1 + z * (1 - p)), torch.zeros_like(z, dtype=torch.bool)
    else:
        y, slope, unsure = z, torch.ones_like(z), torch.zeros_like(z, dtype=torch.bool)
    curved = 1.0 if act == 'silu' else 0.0
    t_y = 1.1 * t_z + curved * 8 * U * y.abs() * (1 + z.abs())
    dz = dy * slope
    t_dz = dy.abs() * (curved * (0.5 * t_z + 16 * U * (1 + z.abs())) + U) + torch.where(unsure, dy.abs(), 0.0)
    d, t_d = dz * ga, t_dz * ga.abs() + U * (dz * ga).abs()
    m1, m2 = whole(gmean(d)), whole(gmean(d * xh))
    t_m1 = whole(gmean(t_d)) + L * U * whole(gmean(d.abs()))
    t_m2 = whole(gmean(t_d * xh.abs() + d.abs() * t_xh)) + L * U * whole(gmean((d * xh).abs()))
    dx = (d - m1 - xh * m2) * rstd
    t_dx = rstd * (t_d + t_m1 + xh.abs() * t_m2 + m2.abs() * t_xh + 4 * U * (d.abs() + m1.abs() + (xh * m2).abs())) + (L + 4) * U * dx.abs()
    t_dx = torch.where(unsure, math.inf, t_dx)
    dgamma, dbeta = (dz * xh).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
    t_dg = (t_dz * xh.abs() + dz.abs() * t_xh).sum(dim=(0, 1)) + 2 * L * U * (dz * xh).abs().sum(dim=(0, 1))
    t_db = t_dz.sum(dim=(0, 1)) + 2 * L * U * dz.abs().sum(dim=(0, 1))  # (twice: within a sample, and over the samples)
    return (y, dx, dgamma, dbeta), (t_y, t_dx, t_dg, t_db)


def _check(got, want, tol, dtype, what):
    got = got.detach().double().reshape(want.shape)
    tol = tol + HALF[dtype] * (want.abs() + tol).clamp(max=1e300) + (2.0**-25 if dtype == torch.float16 else 0.0)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()}, worst {float(((got - want).abs() / tol.clamp(min=1e-300)).max()):.3g} times the tolerance'


def _run(dev, shape, G, dtype, act, seed, eps=1e-3, scale=True, center=True, offset=0.5):
    from hgq2_amd import ops

    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = (torch.randn(shape, generator=g) + offset * torch.randn(C, generator=g)).to(dtype).to(dev).requires_grad_(True)
    dy = torch.randn(shape, generator=g).to(dtype).to(dev)
    gamma = (1 + 0.3 * torch.randn(C, generator=g)).to(dev).requires_grad_(True) if scale else None
    beta = (0.3 * torch.randn(C, generator=g)).to(dev).requires_grad_(True) if center else None
    y = ops.group_norm(x, G, gamma, beta, eps, act)
    assert y.dtype == dtype and y.shape == x.shape
    leaves = [t for t in (x, gamma, beta) if t is not None]
    grads = list(torch.autograd.grad(y, leaves, dy))
    flat = (shape[0], -1, C)
    want, tol = _definition(x.detach().reshape(flat), dy.reshape(flat), None if gamma is None else gamma.detach(), None if beta is None else beta.detach(), G, eps, act)
    _check(y, want[0], tol[0], dtype, 'y')
    _check(grads.pop(0), want[1], tol[1], dtype, 'dx')
    if scale:
        _check(grads.pop(0), want[2], tol[2], torch.float32, 'dgamma')
    if center:
        _check(grads.pop(0), want[3], tol[3], torch.float32, 'dbeta')


# a row of one channel; channels by themselves; whole samples; rows of odd width; groups narrower and wider than 16 bytes; few long and many short samples
SHAPES = [((3, 1, 1), 1), ((1, 7), 7), ((5, 24), 4), ((4, 1, 64), 1), ((2, 9, 33), 3), ((2, 5, 7, 35), 5), ((3, 17, 40), 40), ((2, 6, 6, 32), 8),
          ((2, 1, 30, 48), 6), ((97, 30, 48), 6), ((1, 28, 28, 32), 8), ((2, 64, 64, 64), 1), ((1, 61, 67, 96), 4), ((3, 2, 3, 4, 16), 2),
          ((2, 3, 5000), 1), ((1, 4, 9000), 2), ((2, 100, 1000), 250), ((1, 20000, 8), 2), ((1, 130, 130, 24), 3), ((700, 3, 6), 2), ((2, 300, 512), 32),
          ((1, 5, 8192), 1), ((1, 3, 12288), 3), ((2, 40, 1028), 257), ((1, 70000, 4), 4), ((40, 49, 256), 32), ((1, 1, 100000), 1)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('shape,G', SHAPES)
def test_against_64_bits(dev, shape, G, dtype):
    act = ('linear', 'relu', 'silu')[(sum(shape) + G) % 3]
    _run(dev, shape, G, dtype, act, sum(shape) * 7 + G)


@pytest.mark.parametrize('act', ['linear', 'relu', 'silu', 'swish', None])
@pytest.mark.parametrize('scale,center', [(True, True), (False, True), (True, False), (False, False)])
def test_activations_and_missing_variables(dev, act, scale, center):
    _run(dev, (6, 10, 10, 20), 5, torch.float32, act if act != 'swish' else 'silu', 5, scale=scale, center=center)
    from hgq2_amd import ops

    x = torch.randn(3, 4, 8, device=dev)
    if act in ('swish', None):
        assert torch.equal(ops.group_norm(x, 2, activation=act), ops.group_norm(x, 2, activation={'swish': 'silu', None: 'linear'}[act]))


@pytest.mark.parametrize('shape,G', [((2, 50, 32), 4), ((1, 40000, 16), 2), ((2, 3, 5000), 1)])
def test_far_from_zero(dev, shape, G):
    """A mean of 3000 standard deviations: mean(x^2) - mean(x)^2 would be noise."""
    from hgq2_amd import ops

    g = torch.Generator().manual_seed(2)
    x = (torch.randn(shape, generator=g) + 3000.0).to(dev)
    y = ops.group_norm(x, G, epsilon=0.0)
    # (fp32 holds x to 2^-13 of the standard deviation; the kernel starts from what is held)
    want, tol = _definition(x, torch.zeros(shape), None, None, G, 0.0, 'linear')
    _check(y, want[0], tol[0], torch.float32, 'y')
    assert abs(float(y.double().square().mean()) - 1) < 0.01


def test_what_is_not_finite_stays_in_its_group(dev):
    from hgq2_amd import ops

    for shape, G in (((4, 20, 12), 3), ((2, 50000, 8), 2), ((3, 2, 6000), 2)):
        g = torch.Generator().manual_seed(3)
        x = torch.randn(shape, generator=g).to(dev)
        dy = torch.randn(shape, generator=g).to(dev)
        for bad in (float('nan'), float('inf')):
            for act in ('linear', 'relu', 'silu'):
                outs = []
                for poison in (False, True):
                    xp = x.clone()
                    if poison:
                        xp[1, 1, 0] = bad
                    xp.requires_grad_(True)
                    y = ops.group_norm(xp, G, activation=act)
                    outs.append((y.detach(), *torch.autograd.grad(y, xp, dy)))
                D = shape[-1] // G
                for a, b in zip(*outs):
                    keep = torch.ones(shape, dtype=torch.bool, device=dev)
                    keep[1, :, :D] = False
                    assert torch.equal(a[keep], b[keep]) and torch.isfinite(a).all()
                    assert torch.isnan(b[~keep]).all()


def test_empty_batches(dev):
    from hgq2_amd import ops

    for shape in ((0, 5, 8), (3, 0, 8)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        gamma, beta = torch.ones(8, device=dev, requires_grad=True), torch.zeros(8, device=dev, requires_grad=True)
        y = ops.group_norm(x, 2, gamma, beta)
        dx, dg, db = torch.autograd.grad(y, [x, gamma, beta], torch.zeros(shape, device=dev))
        assert y.shape == dx.shape == shape and not dg.any() and not db.any()


def test_strides_offsets_and_partial_gradients(dev):
    """Views that begin off an aligned address, transposed inputs and gradients, and gradients of some operands only."""
    from hgq2_amd import ops

    g = torch.Generator().manual_seed(4)
    for dtype in (torch.float32, torch.bfloat16):
        for C, G, S in ((32, 8, 50), (32, 8, 20000), (48, 6, 30)):
            buf = torch.randn(1 + 2 * S * C, generator=g).to(dtype).to(dev)
            x = buf[1:].view(2, S, C)
            dy = torch.randn(2, C, S, generator=g).to(dtype).to(dev).transpose(1, 2)
            gamma = torch.randn(1 + C, generator=g).to(dev)[1:]
            xs, ga = x.clone().requires_grad_(True), gamma.clone().requires_grad_(True)
            xt = x.transpose(1, 2).contiguous().transpose(1, 2).requires_grad_(True)
            base = ops.group_norm(xs, G, ga, activation='silu')
            wx, wg = torch.autograd.grad(base, [xs, ga], dy.contiguous())
            xv = x.detach().requires_grad_(True)
            gv = gamma.detach().requires_grad_(True)
            y = ops.group_norm(xv, G, gv, activation='silu')
            vx, vg = torch.autograd.grad(y, [xv, gv], dy)
            tol = 2.0**-7 if dtype == torch.bfloat16 else 1e-5  # (another order of the same sums)
            for a, b in ((y, base), (vx, wx)):
                assert float((a.float() - b.float()).abs().max()) <= tol * float(b.float().abs().max())
            assert float((vg - wg).abs().max()) <= 1e-4 * float(wg.abs().max())
            yt = ops.group_norm(xt, G, ga, activation='silu')
            assert torch.equal(yt, base)
            only_gamma, = torch.autograd.grad(ops.group_norm(x.clone(), G, ga, activation='silu'), [ga], dy.contiguous())
            assert torch.equal(only_gamma, wg)
            only_x, = torch.autograd.grad(ops.group_norm(xs, G, ga.detach(), activation='silu'), [xs], dy.contiguous())
            assert torch.equal(only_x, wx)


def test_gradients_against_differences(dev):
    """Directional differences of the definition in 64 bits at the same point: the error of a central difference of step h is of order
    h^2, 1e-8 here, and the fp32 gradients are within 1e-5 of their scale."""
    from hgq2_amd import ops

    g = torch.Generator().manual_seed(5)
    x0, dy = torch.randn(3, 11, 12, generator=g), torch.randn(3, 11, 12, generator=g)
    ga0, be0 = 1 + 0.3 * torch.randn(12, generator=g), 0.3 * torch.randn(12, generator=g)

    def value(x, ga, be):
        t = x.view(3, 11, 4, 3)
        m = t.mean(dim=(1, 3), keepdim=True)
        v = ((t - m) ** 2).mean(dim=(1, 3), keepdim=True)
        z = ((t - m) / torch.sqrt(v + 1e-3)).reshape(3, 11, 12) * ga + be
        return float((z * torch.sigmoid(z) * dy.double()).sum())

    ops_in = [t.to(dev).requires_grad_(True) for t in (x0, ga0, be0)]
    grads = torch.autograd.grad(ops.group_norm(ops_in[0], 4, ops_in[1], ops_in[2], 1e-3, 'silu'), ops_in, dy.to(dev))
    for k in range(3):
        for trial in range(4):
            at = [t.double() for t in (x0, ga0, be0)]
            way = torch.randn(at[k].shape, generator=g, dtype=torch.float64)
            h = 1e-4
            lo, hi = list(at), list(at)
            lo[k], hi[k] = at[k] - h * way, at[k] + h * way
            diff = (value(*hi) - value(*lo)) / (2 * h)
            have = float((grads[k].double().cpu() * way).sum())
            assert abs(have - diff) <= 1e-5 * float((grads[k].double().cpu() * way).abs().sum()) + 1e-6


@pytest.mark.parametrize('shape,G', [((64, 13, 13, 32), 8), ((2, 128, 128, 32), 4), ((2, 5, 6000), 2)])
def test_recorded_and_repeated(dev, shape, G):
    """Forward and backward recorded together: every replay gives the eager bits for the inputs of its time, and two recordings that are
    replayed in turn do not disturb each other; repeated calls give the same bits."""
    from hgq2_amd import ops

    gen = torch.Generator().manual_seed(6)
    C = shape[-1]
    feeds = [(torch.randn(shape, generator=gen).to(dev), torch.randn(shape, generator=gen).to(dev)) for _ in range(3)]
    gamma, beta = torch.randn(C, generator=gen).to(dev).requires_grad_(True), torch.randn(C, generator=gen).to(dev).requires_grad_(True)

    def both(x, dy):
        y = ops.group_norm(x, G, gamma, beta, activation='relu')
        return (y.detach(), *torch.autograd.grad(y, [x, gamma, beta], dy))

    eager = [both(x.clone().requires_grad_(True), dy) for x, dy in feeds]
    again = both(feeds[0][0].clone().requires_grad_(True), feeds[0][1])
    assert all(torch.equal(a, b) for a, b in zip(eager[0], again))
    side = torch.cuda.Stream()
    recorded = []
    for _ in range(2):
        x, dy = feeds[0][0].clone().requires_grad_(True), feeds[0][1].clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both(x, dy)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = both(x, dy)
        recorded.append((graph, x, dy, out))
    for k in (0, 1, 2, 1, 0):
        for graph, x, dy, _ in recorded:
            with torch.no_grad():
                x.copy_(feeds[k][0]), dy.copy_(feeds[k][1])
        for graph, *_ in recorded:
            graph.replay()
        both(feeds[2][0].clone().requires_grad_(True), feeds[2][1])  # eager work between the replays
        torch.cuda.synchronize()
        for _, _, _, out in recorded:
            assert all(torch.equal(a, b) for a, b in zip(out, eager[k])), k


def test_layer_against_its_host_form(dev):
    from hgq2_amd.host import GroupNormalization

    g = torch.Generator().manual_seed(7)
    x = torch.randn(4, 9, 9, 24, generator=g)
    for act in (None, 'relu', 'silu'):
        layer = GroupNormalization(6, activation=act)
        layer(x.to(dev))
        with torch.no_grad():
            layer.gamma.copy_(torch.rand(24, generator=g) + 0.5), layer.beta.copy_(torch.randn(24, generator=g))
        got, want = layer(x.to(dev), training=True).detach().cpu().double(), layer.host_fn(x.double())
        assert float((got - want).abs().max()) <= 1e-5 * float(want.abs().max())


@pytest.mark.parametrize('bits', [32, 8])
def test_a_normalised_network_trained_with_adamw(dev, bits):
    """The operators together as they are used: a quantized convolution, group normalisation with its activation, a quantized dense layer; loss,
    clipped AdamW step; recorded, against the same steps run eagerly."""
    from hgq2_amd import ops
    from hgq2_amd.config import LayerConfigScope, QuantizerConfigScope
    from hgq2_amd.host import Flatten, GroupNormalization, MaxPooling2D, Sequential
    from hgq2_amd.layers import QConv2D, QDense
    from hgq2_amd.train import AdamW, model_loss, train_step_for

    g = torch.Generator().manual_seed(8)
    x, y = torch.rand(12, 14, 14, 1, generator=g).to(dev), torch.randint(0, 10, (12,), generator=g).to(dev)

    def net():
        with QuantizerConfigScope(place='all', default_q_type='kbi', overflow_mode='SAT_SYM'), \
             QuantizerConfigScope(place='datalane', default_q_type='kif', overflow_mode='WRAP'), LayerConfigScope(enable_ebops=True, beta0=1e-6):
            model = Sequential([QConv2D(16, 3), GroupNormalization(4, activation='relu'), MaxPooling2D((2, 2)), QConv2D(8, 3), GroupNormalization(1, activation='silu'),
                                Flatten(), QDense(10)])
        model(x, training=False)
        return model

    make = lambda v: AdamW(v, lr=0.003, global_clipnorm=2.0, state_bits=bits, seed=3, fold_regularizers=True)  # noqa: E731
    a, b = net(), net()
    with torch.no_grad():
        for p, q in zip(a.parameters(), b.parameters()):
            q.copy_(p)
    names = [p.var_name for p in a.parameters() if p.requires_grad]
    assert names.count('gamma') == 2 and names.count('beta') >= 2
    step = train_step_for(a, x, y, optimizer=make, warmup=1)
    losses = [float(step()) for _ in range(3)]
    opt = make(b.parameters())
    for k in range(4):
        opt.zero_grad()
        loss = model_loss(b, ops.sparse_ce(b(x, training=True), y), True)
        opt.backward(loss)
        opt.step()
        if k:
            assert float(loss) == losses[k - 1]  # the same launches
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q) and torch.isfinite(p).all()
    assert step.opt.iterations == opt.iterations == 4


def test_gradients_of_gradients_are_refused(dev):
    from hgq2_amd import ops

    x = torch.randn(2, 5, 8, device=dev, requires_grad=True)
    y = ops.group_norm(x, 2, activation='silu')
    plain, = torch.autograd.grad(y.sum(), x, retain_graph=True)
    once, = torch.autograd.grad(y.sum(), x, create_graph=True)
    assert torch.equal(once.detach(), plain)
    with pytest.raises(RuntimeError, match='differentiable once'):
        once.sum().backward()


@pytest.mark.parametrize('shape,G,dtype,act', [((1100, 26, 26, 32), 8, torch.float32, 'silu'), ((20, 61, 64, 1024), 32, torch.bfloat16, 'linear')])
def test_more_than_the_cache_holds(dev, shape, G, dtype, act):
    """Tensors whose pass exceeds the card's cache (outputs written past it), by their first and last samples and by the sums over all."""
    from hgq2_amd import ops

    g = torch.Generator(device=dev).manual_seed(9)
    C = shape[-1]
    x = torch.randn(shape, generator=g, device=dev).to(dtype).requires_grad_(True)
    dy = torch.randn(shape, generator=g, device=dev).to(dtype)
    gamma, beta = (1 + 0.3 * torch.randn(C, generator=g, device=dev)).requires_grad_(True), torch.randn(C, generator=g, device=dev).requires_grad_(True)
    y = ops.group_norm(x, G, gamma, beta, 1e-3, act)
    dx, dgamma, dbeta = torch.autograd.grad(y, [x, gamma, beta], dy)
    for part in (slice(0, 3), slice(shape[0] - 3, shape[0])):
        flat = (3, -1, C)
        want, tol = _definition(x[part].detach().reshape(flat), dy[part].reshape(flat), gamma.detach(), beta.detach(), G, 1e-3, act)
        _check(y[part], want[0], tol[0], dtype, 'y')
        _check(dx[part], want[1], tol[1], dtype, 'dx')
    sums, tols = [0, 0], [0, 0]
    for at in range(0, shape[0], 50):
        part = slice(at, at + 50)
        flat = (len(x[part]), -1, C)
        want, tol = _definition(x[part].detach().reshape(flat), dy[part].reshape(flat), gamma.detach(), beta.detach(), G, 1e-3, act)
        for k in range(2):
            sums[k], tols[k] = sums[k] + want[2 + k], tols[k] + tol[2 + k]
    _check(dgamma, sums[0], tols[0], torch.float32, 'dgamma')
    _check(dbeta, sums[1], tols[1], torch.float32, 'dbeta')


def test_what_is_refused_on_the_gpu(dev):
    from hgq2_amd import ops

    x = torch.randn(2, 5, 8, device=dev)
    one = torch.ones(8, device=dev)
    for kw in (dict(groups=3), dict(groups=0), dict(groups=-1), dict(groups=16)):
        with pytest.raises(ValueError, match='groups of one size'):
            ops.group_norm(x, **kw)
    for gamma in (one[:4], one.view(1, 8), torch.empty(0, device=dev), one.cpu(), one.double(), one.bfloat16(), torch.ones(16, device=dev)[::2]):
        with pytest.raises(ValueError, match='gamma'):
            ops.group_norm(x, 2, gamma)
        with pytest.raises(ValueError, match='beta'):
            ops.group_norm(x, 2, one, gamma)
    with pytest.raises(ValueError, match='float32'):
        ops.group_norm(x.double(), 2)
    with pytest.raises(ValueError, match='batch'):
        ops.group_norm(one, 2)
    y, stats = torch.ops.hgq.group_norm_fwd(x, one, one, 2, 1e-3, 0)
    for args in ((x[:1], x, one, one, stats), (x.bfloat16(), x, one, one, stats), (x, x, one, one, stats[:1]), (x.transpose(0, 1), x, one, one, stats)):
        with pytest.raises(ValueError):
            torch.ops.hgq.group_norm_bwd(*args, 2, 0, True, True, True)


def test_two_backward_passes_and_another_stream(dev):
    from hgq2_amd import ops

    g = torch.Generator().manual_seed(10)
    x = torch.randn(40, 300, 64, generator=g).to(dev).requires_grad_(True)
    gamma = torch.randn(64, generator=g).to(dev).requires_grad_(True)
    dy = torch.randn(40, 300, 64, generator=g).to(dev)
    y = ops.group_norm(x, 8, gamma, activation='silu')
    first = torch.autograd.grad(y, [x, gamma], dy, retain_graph=True)
    again = torch.autograd.grad(y, [x, gamma], dy)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = ops.group_norm(x, 8, gamma, activation='silu')
        there = torch.autograd.grad(z, [x, gamma], dy)
    s.synchronize()
    assert torch.equal(y, z) and all(torch.equal(a, b) for a, b in zip(first, there))
    with pytest.raises(RuntimeError, match='modified'):
        w = torch.randn(2, 5, 8, device=dev, requires_grad=True)
        v = w * 1.0
        out = ops.group_norm(v, 2)
        v.add_(1.0)
        out.sum().backward()


# more groups than a launch has workgroups of 256 threads; 67 million groups of one access per row; more than 2^31 elements
@pytest.mark.parametrize('shape,G,dtype', [((129, 2, 131072), 131072, torch.float32), ((16400, 2, 16396), 4099, torch.bfloat16),
                                           ((33, 1 << 16, 1024), 8, torch.bfloat16)])
def test_very_many_groups_and_elements(dev, shape, G, dtype):
    from hgq2_amd import ops

    g = torch.Generator(device=dev).manual_seed(12)
    x = torch.randn(shape, generator=g, device=dev, dtype=dtype).requires_grad_(True)
    dy = torch.randn(shape, generator=g, device=dev, dtype=dtype)
    gamma, beta = (torch.randn(shape[-1], generator=g, device=dev) for _ in range(2))
    y = ops.group_norm(x, G, gamma, beta, activation='silu')
    dx, = torch.autograd.grad(y, x, dy)
    for b in (0, shape[0] // 2, shape[0] - 1):
        part = slice(b, b + 1)
        want, tol = _definition(x[part].detach(), dy[part], gamma, beta, G, 1e-3, 'silu')
        _check(y[part], want[0], tol[0], dtype, f'y of sample {b}')
        _check(dx[part], want[1], tol[1], dtype, f'dx of sample {b}')


def test_recording_while_another_streams_graph_lives(dev):
    """A leaf whose gradients an earlier, living graph of another stream accumulates is refused in a recording, and taken once that is gone."""
    from hgq2_amd import ops

    g = torch.Generator().manual_seed(13)
    x = torch.randn(4, 20, 16, generator=g).to(dev)
    gamma = torch.nn.Parameter(torch.randn(16, generator=g).to(dev))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # outside a recording either stream will do
        want = torch.autograd.grad(ops.group_norm(x, 4, gamma).square().sum(), gamma)[0]
    torch.cuda.synchronize()
    living = ops.group_norm(x, 4, gamma)
    with pytest.raises(RuntimeError, match='gamma belongs to a graph of another stream'):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            ops.group_norm(x, 4, gamma)
    del living
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.group_norm(x, 4, gamma).backward(2 * ops.group_norm(x, 4, gamma.detach()))
    got = gamma.grad
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)


def test_tangents_are_refused_and_a_call_without_gradients_makes_no_node(dev):
    import torch.autograd.forward_ad as fw

    from hgq2_amd import ops

    x = torch.randn(2, 5, 8, device=dev)
    gamma = torch.nn.Parameter(torch.ones(8, device=dev))
    y = ops.group_norm(x, 2, gamma)
    with torch.no_grad():
        z = ops.group_norm(x, 2, gamma)
    assert y.requires_grad and not z.requires_grad and torch.equal(y, z) and not ops.group_norm(x, 2).requires_grad
    with fw.dual_level(), pytest.raises(Exception, match='jvp|forward'):
        ops.group_norm(fw.make_dual(x, torch.ones_like(x)), 2)


def test_two_threads(dev):
    """Two threads, each on a stream of its own, get what one gets alone."""
    import threading

    from hgq2_amd import ops

    g = torch.Generator().manual_seed(17)
    data = []
    for shape, G in (((50, 100, 48), 6), ((3, 5000, 32), 4)):
        data.append((torch.randn(shape, generator=g).to(dev).requires_grad_(True), torch.randn(shape[-1], generator=g).to(dev).requires_grad_(True), G,
                     torch.randn(shape, generator=g).to(dev)))

    def work(x, gamma, G, dy):
        y = ops.group_norm(x, G, gamma, activation='silu')
        return [y.detach(), *torch.autograd.grad(y, [x, gamma], dy), ops.global_norm([y.detach(), dy])]

    want, got = [work(*d) for d in data], [None, None]
    torch.cuda.synchronize()

    def run(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                out = work(*data[k])
            torch.cuda.current_stream().synchronize()
            got[k] = out

    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for a, b in zip(want, got):
        assert b is not None and all(torch.equal(p, q) for p, q in zip(a, b))


def test_recording_again_and_beside_a_living_loss(dev):
    """A second recording of one model works; one beside the living loss of an eager step is refused and leaves everything usable."""
    from hgq2_amd import ops
    from hgq2_amd.config import LayerConfigScope, QuantizerConfigScope
    from hgq2_amd.host import GroupNormalization, Sequential
    from hgq2_amd.layers import QDense
    from hgq2_amd.train import AdamW, model_loss, train_step_for

    g = torch.Generator().manual_seed(19)
    x, y = torch.rand(64, 12, generator=g).to(dev), torch.randint(0, 5, (64,), generator=g).to(dev)
    with QuantizerConfigScope(place='all', default_q_type='kbi', overflow_mode='SAT_SYM'), \
         QuantizerConfigScope(place='datalane', default_q_type='kif', overflow_mode='WRAP'), LayerConfigScope(enable_ebops=True, beta0=1e-6):
        model = Sequential([QDense(24), GroupNormalization(3, activation='relu'), QDense(5)])
    make = lambda v: AdamW(v, lr=0.003, fold_regularizers=True)  # noqa: E731
    for _ in range(2):
        step = train_step_for(model, x, y, optimizer=make)
        assert all(math.isfinite(float(step())) for _ in range(3)) and step.opt.iterations == 6
    opt = make(model.parameters())
    loss = model_loss(model, ops.sparse_ce(model(x, training=True), y), True)
    opt.backward(loss)
    opt.step()
    with pytest.raises(RuntimeError, match='belongs to a graph of another stream'):
        train_step_for(model, x, y, optimizer=make)
    del loss
    step = train_step_for(model, x, y, optimizer=make)
    assert all(math.isfinite(float(step())) for _ in range(3)) and step.opt.iterations == 6


# tiles of which some rows lie in LDS: groups of whole accesses and others, rows of two and four positions with a short last one, 8 and 4 wavefronts
@pytest.mark.parametrize('act', ['linear', 'relu', 'silu'])
@pytest.mark.parametrize('shape,G,dtype', [((600, 26, 26, 32), 8, torch.float32), ((520, 551, 30), 10, torch.float32), ((513, 26, 26, 32), 4, torch.bfloat16),
                                           ((520, 681, 27), 9, torch.float16), ((520, 26, 26, 64), 8, torch.float16), ((512, 360, 32), 4, torch.float32),
                                           ((512, 20, 1024), 1024, torch.float32), ((512, 20, 1024), 512, torch.float32)])
def test_rows_in_lds(dev, shape, G, dtype, act):
    _run(dev, shape, G, dtype, act, sum(shape) + G)


@pytest.mark.parametrize('shape,dtype', [((1024, 26, 26, 32), torch.float32), ((2, 30000, 32), torch.float32), ((40, 30, 48), torch.float16), ((2, 3, 5000), torch.float32)])
def test_the_side_of_a_relus_border(dev, shape, dtype):
    """x next to where z is zero, to both sides, for gammas of both signs and zero: with dy = 1, dx shows what passes.  In 64 bits from the statistics
    that the operator reports, so no rounding but theirs counts."""
    g = torch.Generator().manual_seed(21)
    C, G = shape[-1], 2
    from hgq2_amd import _lib

    _lib.native()
    x = torch.randn(shape, generator=g).to(dtype).to(dev)
    gamma, beta = torch.randn(C, generator=g).to(dev), 0.5 * torch.randn(C, generator=g).to(dev)
    gamma[3], gamma[4], beta[3], beta[4] = 0.0, 0.0, 0.7, -0.7
    for _ in range(3):  # (moving elements to the border moves the statistics a little: again)
        y, stats = torch.ops.hgq.group_norm_fwd(x, gamma, beta, G, 1e-3, 1)
        flat = x.view(shape[0], -1, C)
        mean, rstd = (t.view(shape[0], 1, G).repeat_interleave(C // G, dim=2) for t in stats)
        at = (mean - beta.double() / (gamma.double() * rstd)).to(dtype)
        for k in range(min(3, flat.shape[1])):
            row = at[:, 0] if k == 0 else torch.nextafter(at[:, 0].float(), torch.full_like(at[:, 0].float(), math.inf if k == 1 else -math.inf)).to(dtype)
            flat[:, k] = torch.where(torch.isfinite(row), row, flat[:, k])
    y, stats = torch.ops.hgq.group_norm_fwd(x, gamma, beta, G, 1e-3, 1)
    mean, rstd = (t.view(shape[0], 1, G).repeat_interleave(C // G, dim=2) for t in stats)
    passes = (x.view(shape[0], -1, C).double() - mean) * rstd * gamma.double() + beta.double() > 0
    assert passes[..., 3].all() and not passes[..., 4].any()
    dy = torch.ones_like(x)
    _, _, dbeta = torch.ops.hgq.group_norm_bwd(dy, x, gamma, beta, stats, G, 1, True, True, True)
    assert torch.equal(dbeta.double(), passes.sum(dim=(0, 1)).double())  # (counts below 2^24 are exact)
