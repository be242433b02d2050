"""Norms around a residual sum against their definition in 64 bits.

Tolerances, u = 2^-24 (half a step of fp32).  A row's sum adds eight terms one after the other and goes on pairwise in at most ten levels: 18 u of the
magnitudes, K = 20 with the division.  So r = 1 / sqrt(mean + eps) is relatively off by K / 2 + 3 (root, quotient) u and by what the values under it are off;
every product adds u.  A sigmoid in fp32 is off by (1.5 |g| + 4) u (1 - s) + 2 u relatively.  Sums over rows: a thread adds its rows one after the other
(fewer than 64 in these tests), up to 256 teams meet one after the other, 64 bits join the rest: L = 330 u of the magnitudes.  A 16-bit type adds half a step."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U, K, L = 2.0**-24, 20, 330
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LEAST = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25}


def _definition(x, u, gate, post, pre, dy, dh, act, scale, eps):
    """(values, tolerances) of y, h, dx, du, dgate, dpost, dpre; rows [R, C], gate already repeated for each row (its sum is the caller's)."""
    x, dy, dh = x.double(), dy.double(), dh.double()
    ga = pre.double() if pre is not None else torch.ones(x.shape[1], dtype=torch.float64)
    mean = lambda t: t.mean(dim=1, keepdim=True)  # noqa: E731
    if u is not None:
        u = u.double()
        po = (post.double() if post is not None else torch.ones(x.shape[1], dtype=torch.float64)) * scale
        g = None if gate is None else gate.double()
        open_ = torch.ones_like(x) if g is None else torch.sigmoid(g) if act else g
        e_open = torch.zeros_like(x) if g is None or not act else ((1.5 * g.abs() + 4) * (1 - open_) + 2) * U
        r_u = 1 / torch.sqrt(mean(u * u) + eps)
        e_r = (K / 2 + 3) * U
        n = u * r_u
        b = n * po * open_
        y = x + b
        t_y = b.abs() * (e_r + 5 * U + e_open) + 2 * U * y.abs()
    else:
        y, t_y = x, torch.zeros_like(x)
    square = mean(y * y) + eps
    r = 1 / torch.sqrt(square)
    e_y = (K / 2 + 3) * U + 1.1 * mean(y.abs() * t_y) / square.clamp(min=1e-300)
    m = y * r
    t_m = r * t_y + m.abs() * (e_y + 2 * U)
    h, t_h = m * ga, t_m * ga.abs() + 2 * U * (m * ga).abs()
    e, t_e = dh * ga, U * (dh * ga).abs()
    s1 = mean(e * m)
    t_s1 = mean(t_e * m.abs() + e.abs() * t_m) + (K + 2) * U * mean((e * m).abs())
    back = r * (e - m * s1)
    dx = dy + back
    t_dx = r * (t_e + t_m * s1.abs() + m.abs() * t_s1 + 4 * U * (e.abs() + (m * s1).abs())) + (e_y + 2 * U) * back.abs() + 2 * U * (dy.abs() + dx.abs())
    out = dict(y=(y, t_y), h=(h, t_h), dx=(dx, t_dx))
    out['dpre'] = ((dh * m).sum(0), (dh.abs() * t_m + 2 * U * (dh * m).abs()).sum(0) + L * U * (dh * m).abs().sum(0))
    if u is None:
        return out
    db = dx * open_
    t_db = t_dx * open_.abs() + db.abs() * (e_open + 2 * U)
    t_n = n.abs() * (e_r + 2 * U)
    dn, t_dn = db * po, t_db * po.abs() + 3 * U * (db * po).abs()
    s2 = mean(dn * n)
    t_s2 = mean(t_dn * n.abs() + dn.abs() * t_n) + (K + 2) * U * mean((dn * n).abs())
    du = r_u * (dn - n * s2)
    t_du = r_u * (t_dn + t_n * s2.abs() + n.abs() * t_s2 + 4 * U * (dn.abs() + (n * s2).abs())) + (e_r + 2 * U) * du.abs()
    out['du'] = (du, t_du)
    term = db * n * scale
    t_term = (t_db * n.abs() + db.abs() * t_n) * abs(scale) + 3 * U * term.abs()
    out['dpost'] = (term.sum(0), t_term.sum(0) + L * U * term.abs().sum(0))
    if g is not None:
        slope = open_ * (1 - open_) if act else torch.ones_like(x)
        t_slope = slope * (e_open * 2 + (e_open * open_ / (1 - open_).clamp(min=1e-300)) + 6 * U) + 2 * U * open_ if act else torch.zeros_like(x)
        base = n * po
        dg = dx * base * slope
        t_dg = t_dx * (base * slope).abs() + dx.abs() * (base.abs() * t_slope + slope * (t_n * po.abs() + 3 * U * base.abs())) + 4 * U * dg.abs()
        out['dgate'] = (dg, t_dg)
    return out


def _check(got, want, dtype, what):
    want, tol = want
    got = got.detach().double().cpu().reshape(want.shape)
    tol = tol + HALF[dtype] * (want.abs() + tol) + LEAST[dtype]
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()}, worst {float(((got - want).abs() / tol)[bad].max()):.3g} times the tolerance'


def _inputs(shape, dtype, gate, seed, gammas=True):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = (torch.randn(shape, generator=g) * (1 + 3 * torch.rand(C, generator=g))).to(dtype)
    u = (0.3 * torch.randn(shape, generator=g) + 0.1).to(dtype)
    where = {'none': None, 'element': shape, 'sample': (shape[0], C), 'sample_axes': (shape[0], *[1] * (len(shape) - 2), C), 'channel': (C,)}[gate]
    gt = None if where is None else torch.randn(where, generator=g).to(dtype)
    post, pre = ((1 + 0.3 * torch.randn(C, generator=g)) if gammas else None for _ in range(2))
    return x, u, gt, post, pre, torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)


def _repeated(gate, x):
    if gate is None:
        return None
    C = x.shape[-1]
    if gate.shape == x.shape:
        return gate.reshape(-1, C)
    if gate.dim() == 1:
        return gate.expand(x.numel() // C, C)
    return gate.reshape(x.shape[0], 1, C).expand(x.shape[0], x.numel() // C // x.shape[0], C).reshape(-1, C)


def _run(dev, shape, dtype, gate, act, seed, scale=0.75, eps=1e-6, gammas=True):
    from hgq2_amd import ops

    x, u, gt, post, pre, dy, dh = _inputs(shape, dtype, gate, seed, gammas)
    leaves = [None if t is None else t.to(dev).requires_grad_(True) for t in (x, u, gt, post, pre)]
    y, h = ops.residual_norm(leaves[0], leaves[1], leaves[3], leaves[4], leaves[2], act, scale, eps)
    assert y.dtype == h.dtype == dtype and y.shape == h.shape == x.shape
    grads = torch.autograd.grad([y, h], [t for t in leaves if t is not None], [dy.to(dev), dh.to(dev)])
    C = shape[-1]
    flat = lambda t: t.reshape(-1, C)  # noqa: E731
    want = _definition(flat(x), flat(u), _repeated(gt, x), post, pre, flat(dy), flat(dh), act == 'sigmoid', scale, eps)
    if gt is not None and gt.shape != x.shape:  # the sum over the rows that a gate stands for
        dg, t_dg = want['dgate']
        rows = (-1, dg.shape[0] // (gt.numel() // C), C)
        want['dgate'] = (dg.reshape(rows).sum(1), t_dg.reshape(rows).sum(1) + L * U * dg.abs().reshape(rows).sum(1))
    _check(y, want['y'], dtype, 'y')
    _check(h, want['h'], dtype, 'h')
    names = [n for n, t in zip(('dx', 'du', 'dgate', 'dpost', 'dpre'), leaves) if t is not None]
    for name, got, leaf in zip(names, grads, [t for t in leaves if t is not None]):
        assert got.shape == leaf.shape and got.dtype == leaf.dtype
        _check(got, want[name], leaf.dtype, name)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(ops.residual_norm(leaves[0], leaves[1], leaves[3], leaves[4], leaves[2], act, scale, eps), (y, h)))


# one channel; teams of 1 to 64 threads, of 2 to 16 wavefronts, at their borders; odd rows; rows that no workgroup holds; many and few of them
SHAPES = [(1, 1), (3, 2), (700, 7), (5, 8), (6, 3, 9), (4, 33), (2, 300, 64), (31, 30, 48), (2, 3, 5, 100), (17, 333), (40, 512), (9, 513), (3, 7, 1000), (12, 1025), (5, 2049), (2, 4, 4096), (3, 4099),
          (3, 7000), (4, 8192), (2, 2, 8193), (3, 9001), (1, 20000), (4000, 16), (300, 1024)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('shape', SHAPES)
def test_against_64_bits(dev, shape, dtype):
    k = sum(shape)
    gates = ['none', 'element'] + (['sample', 'sample_axes'] if len(shape) > 2 else ['channel'])
    for j in range(2):
        _run(dev, shape, dtype, gates[(k + j) % len(gates)], (None, 'sigmoid')[(k // 2 + j) % 2], k + j, scale=(0.75, -1.0)[j], gammas=bool((k + j) % 3))


@pytest.mark.parametrize('gate', ['none', 'element', 'sample', 'sample_axes', 'channel'])
@pytest.mark.parametrize('act', [None, 'linear', 'sigmoid'])
@pytest.mark.parametrize('shape', [(5, 70, 40), (3, 2, 9, 200), (2, 500, 16), (1500, 3, 24), (2, 40, 1300), (2, 3, 8200), (1, 1, 12)])
def test_gates(dev, shape, act, gate):
    _run(dev, shape, torch.float32, gate, act, len(shape) * 5 + sum(shape))


@pytest.mark.parametrize('gate', ['none', 'element', 'sample'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_several_rows_of_a_workgroup_that_keeps_its_sums_in_lds_or_memory(dev, dtype, gate):
    _run(dev, (2, 300, 4600), dtype, gate, 'sigmoid', 31)
    _run(dev, (2, 150, 8300), dtype, gate, None, 32)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', [(1, 1), (50, 12), (3, 5, 77), (700, 64), (9, 2000), (2, 8200)])
def test_the_norm_by_itself(dev, shape, dtype):
    from hgq2_amd import ops

    for gammas in (True, False):
        x, _, _, _, pre, _, dh = _inputs(shape, dtype, 'none', sum(shape), gammas)
        xd, pd = x.to(dev).requires_grad_(True), pre.to(dev).requires_grad_(True) if gammas else None
        h = ops.rms_norm(xd, pd, 1e-5)
        grads = torch.autograd.grad(h, [t for t in (xd, pd) if t is not None], dh.to(dev))
        flat = lambda t: t.reshape(-1, shape[-1])  # noqa: E731
        want = _definition(flat(x), None, None, None, pre, flat(torch.zeros_like(dh)), flat(dh), False, 1.0, 1e-5)
        _check(h, want['h'], dtype, 'h')
        _check(grads[0], want['dx'], dtype, 'dx')
        if gammas:
            _check(grads[1], want['dpre'], torch.float32, 'dgamma')


def test_one_of_the_outputs_alone(dev):
    """The last block of a network uses h alone, a residual stream without a further norm y alone."""
    from hgq2_amd import ops

    x, u, gt, post, pre, dy, dh = _inputs((6, 9, 50), torch.float32, 'element', 3)
    for use in ('y', 'h'):
        leaves = [t.to(dev).requires_grad_(True) for t in (x, u, gt, post, pre)]
        y, h = ops.residual_norm(leaves[0], leaves[1], leaves[3], leaves[4], leaves[2], 'sigmoid')
        grads = torch.autograd.grad(y if use == 'y' else h, leaves, (dy if use == 'y' else dh).to(dev), allow_unused=True)
        zero = torch.zeros_like(dy)
        flat = lambda t: t.reshape(-1, 50)  # noqa: E731
        want = _definition(flat(x), flat(u), flat(gt), post, pre, flat(dy if use == 'y' else zero), flat(dh if use == 'h' else zero), True, 1.0, 1e-6)
        for name, got, leaf in zip(('dx', 'du', 'dgate', 'dpost', 'dpre'), grads, leaves):
            _check(got, want[name], leaf.dtype, name)


def test_some_of_the_gradients_alone(dev):
    from hgq2_amd import ops

    for shape in ((4, 6, 40), (2, 3, 1500), (2, 2, 9000)):
        x, u, gt, post, pre, dy, dh = _inputs(shape, torch.float32, 'sample', 5)
        tensors = [t.to(dev) for t in (x, u, gt, post, pre)]

        def grads(wanted):
            leaves = [t.clone().requires_grad_(w) for t, w in zip(tensors, wanted)]
            out = ops.residual_norm(leaves[0], leaves[1], leaves[3], leaves[4], leaves[2])
            return torch.autograd.grad(out, [t for t in leaves if t.requires_grad], [dy.to(dev), dh.to(dev)])

        whole = grads([True] * 5)
        for k in range(5):
            (one,) = grads([j == k for j in range(5)])
            assert torch.equal(one, whole[k]), k


def test_against_differences(dev):
    """Along a direction v with entries below 2^-4 the outputs are smooth: a central difference of h = 1 is off by the third derivative / 6.  Inputs of magnitude one
    and rows of 16: a norm's third derivative along v is below 30 |v|^3 rms (bounded by 15 of each factor), with |v| <= 2^-4 per element."""
    from hgq2_amd import ops

    shape = (3, 16)
    g = torch.Generator().manual_seed(7)
    make = lambda *s: (torch.rand(s, generator=g) + 0.5) * torch.where(torch.rand(s, generator=g) < 0.5, -1.0, 1.0)  # noqa: E731
    t = dict(x=make(*shape), u=make(*shape), post=make(16), pre=make(16), gate=make(*shape))
    dy, dh = make(*shape), make(*shape)

    def value(p):
        y, h = ops.residual_norm(p['x'], p['u'], p['post'], p['pre'], p['gate'], 'sigmoid')
        return y, h

    leaves = {k: v.to(dev).requires_grad_(True) for k, v in t.items()}
    grads = dict(zip(t, torch.autograd.grad(value(leaves), list(leaves.values()), [dy.to(dev), dh.to(dev)])))
    for k in t:
        for s in range(3):
            v = (torch.rand(t[k].shape, generator=torch.Generator().manual_seed(s)) * 2 - 1) * 2.0**-4
            hi, lo = (value({**{n: w.to(dev) for n, w in t.items()}, k: (t[k] + f * v).to(dev)}) for f in (1, -1))
            slope = sum(float(((a - b).double().cpu() / 2 * d.double()).sum()) for a, b, d in zip(hi, lo, (dy, dh)))
            tol = 30 * 2.0**-12 / 6 * float(dy.abs().sum() + dh.abs().sum()) + 100 * U * float(dy.abs().sum() + dh.abs().sum())
            assert abs(slope - float((grads[k].double().cpu() * v.double()).sum())) <= tol, k


def test_layouts_of_the_callers(dev):
    """Strided inputs and gradients are taken as they are meant, a gate of float32 for bfloat16 rows is refused."""
    from hgq2_amd import ops

    x, u, gt, post, pre, dy, dh = (None if t is None else t.to(dev) for t in _inputs((6, 10, 24), torch.bfloat16, 'sample', 9))
    want = ops.residual_norm(x, u, post, pre, gt)
    wide = torch.cat([x, x], 2)[..., :24]
    got = ops.residual_norm(wide, u.transpose(0, 1).contiguous().transpose(0, 1), post, torch.stack([pre, pre], 1)[:, 0], torch.stack([gt, gt], 1)[:, 0])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match='gate'):
        ops.residual_norm(x, u, post, pre, gt.float())
    with pytest.raises(ValueError, match='update'):
        ops.residual_norm(x, u.float(), post, pre)


def test_rows_of_zeros_and_large_rows(dev):
    from hgq2_amd import ops

    x = torch.zeros(3, 40, device=dev)
    y, h = ops.residual_norm(x, x)
    assert not y.any() and not h.any()
    y, h = ops.residual_norm(x, x, epsilon=0.0)  # 0 / 0
    assert y.isnan().all() and h.isnan().all()
    small = torch.full((2, 64), 2.0**-66, device=dev)  # squares below fp32's normal numbers, of a few bits each, here exact
    assert torch.equal(ops.rms_norm(small, epsilon=0.0), torch.ones_like(small))
    big = torch.full((2, 64), 2.0**15, dtype=torch.float16, device=dev)  # squares beyond fp16
    assert torch.equal(ops.rms_norm(big), torch.ones_like(big))
    x[1, 3] = float('nan')
    h = ops.rms_norm(x)
    assert h[1].isnan().all() and not h[[0, 2]].any()


@pytest.mark.parametrize('gate', ['none', 'element', 'sample', 'channel'])
def test_no_rows(dev, gate):
    from hgq2_amd import ops

    x, u, gt, post, pre, dy, dh = (None if t is None else t.to(dev).requires_grad_(True) for t in _inputs((0, 3, 12), torch.float32, gate, 1))
    y, h = ops.residual_norm(x, u, post, pre, gt)
    assert y.shape == h.shape == x.shape
    grads = torch.autograd.grad([y, h], [t for t in (x, u, gt, post, pre) if t is not None], [dy, dh])
    assert all(g is not None and not g.any() for g in grads)
    assert ops.rms_norm(x, pre).shape == x.shape


def test_more_than_a_launch_of_samples(dev):
    """70 000 samples of a gate each, in runs that are joined: one launch takes 65 535 of them."""
    from hgq2_amd import ops

    x, u, gt, post, pre, dy, dh = (t.to(dev) for t in _inputs((70000, 3, 8), torch.float32, 'sample', 21))
    leaf = gt.clone().requires_grad_(True)
    (dg,) = torch.autograd.grad(ops.residual_norm(x, u, post, pre, leaf)[0], [leaf], dy)
    n = u.double() / torch.sqrt((u.double()**2).mean(-1, keepdim=True) + 1e-6) * post.double()
    want = (dy.double() * n).sum(1)
    assert ((dg.double() - want).abs() <= 40 * U * (dy.double() * n).abs().sum(1)).all()


def test_recorded_and_on_another_stream(dev):
    from hgq2_amd import ops

    for shape, gate in (((5, 40, 48), 'sample'), ((3, 1500), 'element')):
        feeds = [[t.to(dev) for t in _inputs(shape, torch.bfloat16, gate, s)] for s in range(3)]

        def both(x, u, gt, post, pre, dy, dh):
            y, h = ops.residual_norm(x, u, post, pre, gt, 'sigmoid')
            return (y.detach(), h.detach(), *torch.autograd.grad([y, h], [x, u, gt, post, pre], [dy, dh]))

        leaves = lambda f: [t.clone().requires_grad_(k < 5) for k, t in enumerate(f)]  # noqa: E731
        eager = [both(*leaves(f)) for f in feeds]
        side, recorded = torch.cuda.Stream(), []
        for _ in range(2):
            mine = leaves(feeds[0])
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                first = both(*mine)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(first, eager[0]))
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = both(*mine)
            recorded.append((graph, mine, out))
        for k in (0, 1, 2, 1):
            for _, mine, _ in recorded:
                with torch.no_grad():
                    for a, b in zip(mine, feeds[k]):
                        a.copy_(b)
            for graph, *_ in recorded:
                graph.replay()
            both(*leaves(feeds[2]))
            torch.cuda.synchronize()
            for _, _, out in recorded:
                assert all(torch.equal(a, b) for a, b in zip(out, eager[k])), k


def test_recording_beside_a_living_graph_is_refused_and_gradients_are_not_differentiated(dev):
    from hgq2_amd import ops

    x, p = torch.randn(4, 8, device=dev), torch.nn.Parameter(torch.ones(8, device=dev))
    living = ops.residual_norm(x, x, pre_gamma=p)
    side = torch.cuda.Stream()
    with pytest.raises(RuntimeError, match='pre_gamma belongs to a graph of another stream'):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            ops.residual_norm(x, x, pre_gamma=p)
    (d,) = torch.autograd.grad(living[1].square().sum(), [p], create_graph=True)
    with pytest.raises(RuntimeError, match='differentiable once'):
        d.sum().backward()
    with torch.no_grad():
        assert not ops.residual_norm(x, x, pre_gamma=p)[1].requires_grad


def test_rows_of_a_gate_that_is_not_there(dev):
    """The operators take the rows that a gate's row stands for as a number, which says nothing without a gate."""
    g = torch.Generator().manual_seed(29)
    none = torch.empty(0, device=dev)
    for C in (40, 700, 9000):
        x, u, dy, dh = (torch.randn(24, C, generator=g).to(dev) for _ in range(4))
        got = []
        for P in (1, 6):
            y, h, r = torch.ops.hgq.residual_norm_fwd(x, u, none, none, None, P, 0.5, 1e-6, 0)
            got.append([y, h, r, *torch.ops.hgq.residual_norm_bwd(dy, dh, x, u, none, none, None, r, P, 0.5, 1e-6, 0, True, True, False, True, True)])
        assert all(torch.equal(a, b) for a, b in zip(*got))
