"""The loss against a teacher's top logits, and its gradient, against its definition in 64 bits.

Tolerances, u = 2^-24 (half a step of fp32).  exp(d / T) in fp32, d = z - max: the difference is off by u |d|, the product with 1 / (T ln 2) by
u |d| / T (in two pieces for float32 logits, which only makes it less), the exponential by 2 u, so relatively by (4 + 4 D) u with D the largest |d| / T.  A
sum of a row adds at most 64 terms one after the other and goes on pairwise in at most 32 levels: 96 u more.  So q is relatively off by
E = (120 + 8 D) u, a logarithm of q absolutely by as much, p likewise (D of the teacher's list), 1 - sum p absolutely by E.  The gradient
c (P q - p - p' q / q') then by |c| (2 E P q + E p + 2 E share + E q / q') + 4 u of each, the loss by T^2 sum (p E (|log p - log q| + 2)) + E (|log p' / q'| + 2).
A 16-bit type adds half a step of the result, and of what fp16 holds below its normal numbers."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LEAST = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25}


def _definition(z, t, i, T, lse, w, up=1.0):
    """Loss, gradient and their tolerances, in 64 bits, row by row."""
    z, t = z.double(), t.double()
    N, V = z.shape
    loss, tol = 0.0, 0.0
    grad, gtol = torch.zeros_like(z), torch.zeros_like(z)
    for r in range(N):
        weight = 1.0 if w is None else float(w[r])
        ok = (i[r] >= 0) & (i[r] < V)
        ids, tr = i[r][ok].long(), t[r][ok] / T
        if weight == 0 or not len(ids) or float(tr.max()) == -math.inf:
            continue
        zr = z[r] / T
        log_q = zr - torch.logsumexp(zr, 0)
        q = log_q.exp()
        p = (tr - (torch.logsumexp(tr, 0) if lse is None else float(lse[r]))).exp()
        finite = zr[zr > -math.inf]
        D = max(float(finite.max() - finite.min()), float((tr[tr > -math.inf].max() - tr[tr > -math.inf].min())) if len(ids) else 0.0)
        E = (120 + 8 * D) * U
        at = torch.zeros(V, dtype=torch.float64).index_add_(0, ids, p)
        listed = torch.zeros(V, dtype=torch.bool).index_fill_(0, ids, True)
        terms = torch.where(p > 0, p * (p.clamp(min=1e-300).log() - log_q[ids]), torch.zeros_like(p))
        row, rtol = float(terms.sum()), E * float((torch.where(p > 0, (p.clamp(min=1e-300).log() - log_q[ids]).abs(), torch.zeros_like(p)) * p).sum() + 2 * p.sum())
        rest, share, P = 0.0, torch.zeros_like(q), float(p.sum())
        st = torch.zeros_like(q)
        if lse is not None:
            q_rest = float(q[~listed].sum())
            if q_rest > 0:
                rest = max(0.0, 1.0 - P)
                share = torch.where(listed, torch.zeros_like(q), q / q_rest)
                if rest > 0:
                    row += rest * (math.log(rest) - math.log(q_rest))
                    rtol += E * (abs(math.log(rest / q_rest)) + 2)
                else:
                    rtol += E * (abs(math.log(q_rest)) + 30)
                st = E * share
        c = up * weight * T / N
        loss += weight * T * T / N * row
        tol += abs(weight) * T * T / N * rtol
        grad[r] = c * (q * (P + rest) - at - share * rest)
        gtol[r] = abs(c) * (2 * E * q * (P + rest) + 2 * E * at + 2 * E * share * rest + st + 4 * U * (q + at + share * rest))
    return loss, tol + 4 * U * abs(loss), grad, gtol


def _inputs(rows, V, K, dtype, seed, T=2.0, rest=False, weights=False, index=torch.int64, missing=True, masked=0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn((rows, V), generator=g) * 2 * T).to(dtype)
    if masked:
        z[:, V - masked:] = -math.inf
    i = torch.stack([torch.randperm(V, generator=g)[:K] if K <= V else torch.randint(0, V, (K,), generator=g) for _ in range(rows)])
    t = (torch.randn((rows, K), generator=g) * 2 * T + 4 * T).to(dtype)
    if masked:
        i = torch.where(i >= V - masked, -1, i)
    if missing and rows > 2:
        i[1, K // 2:] = -1
        i[2] = -1
        i[0, 0] = V + 3  # not one of the vocabulary either
    lse = (torch.logsumexp(t.double() / T, 1) + 0.3 * torch.rand(rows, generator=g, dtype=torch.float64)).float() if rest else None
    w = torch.rand(rows, generator=g) - 0.2 if weights else None
    if weights and rows > 3:
        w[3] = 0.0
    return z, t, i.to(index), lse, w


def _check(got, want, tol, dtype, what):
    got = got.detach().double().cpu()
    tol = tol + HALF[dtype] * (want.abs() + tol) + LEAST[dtype]
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()}, worst {float(((got - want).abs() / tol)[bad].max()):.3g} times the tolerance'


def _on(dev, *tensors):
    return [None if t is None else t.to(dev) for t in tensors]


def _run(dev, args, T, dtype, up=None):
    from hgq2_amd import ops

    z, t, i, lse, w = args
    zd, td, id_, ld, wd = _on(dev, z, t, i, lse, w)
    zd.requires_grad_(True)
    loss = ops.distill_topk(zd, td, id_, T, ld, wd)
    assert loss.dtype == torch.float32 and loss.shape == ()
    (dz,) = torch.autograd.grad(loss * up if up is not None else loss, [zd])
    assert dz.dtype == dtype and dz.shape == z.shape
    want = _definition(z, t, i, T, lse, w, 1.0 if up is None else up)
    assert abs(float(loss) - want[0]) <= want[1], (float(loss), want[:2])
    _check(dz, want[2], want[3], dtype, 'dz')
    with torch.no_grad():
        assert float(ops.distill_topk(zd, td, id_, T, ld, wd)) == float(loss)


# one entry; a list as long as the vocabulary; teams of 8, 64, 256 and 1024 threads at their borders, rows that are read twice, rows in parts
SIZES = [(1, 1, 1), (5, 2, 1), (7, 5, 5), (33, 64, 64), (9, 65, 3), (4, 64, 65), (6, 2048, 50), (5, 2049, 700), (4, 7001, 20), (3, 16385, 64), (260, 9000, 10), (257, 17000, 5),
         (256, 65537, 8), (1, 8192, 100), (2, 50001, 33), (1, 300001, 1000)]


# one type for the largest
@pytest.mark.parametrize('rows,V,K,dtype', [(*s, t) for s in SIZES for t in (torch.float32, torch.bfloat16, torch.float16)
                                            if s[0] * s[1] <= 2_000_000 or t == (torch.bfloat16 if s[1] % 2 else torch.float32)])
def test_against_64_bits(dev, rows, V, K, dtype):
    many = rows * V > 2_000_000
    for k, rest in enumerate((False, True)):
        args = _inputs(rows, V, K, dtype, rows + V + K, rest=rest, weights=bool((rows + k) % 2), index=(torch.int32, torch.int64)[k], masked=V // 50 if V > 100 and not many else 0)
        _run(dev, args, 2.0, dtype)


@pytest.mark.parametrize('T', [0.25, 0.7, 1.0, 8.0])
@pytest.mark.parametrize('rest', [False, True])
def test_temperatures(dev, T, rest):
    _run(dev, _inputs(6, 333, 17, torch.float32, 3, T=T, rest=rest), T, torch.float32)


@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('up', [-3.0, 0.0, 1024.0])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_another_upstream_gradient(dev, up, rest, dtype):
    _run(dev, _inputs(37, 500, 9, dtype, 5, rest=rest, weights=True), 2.0, dtype, up)
    _run(dev, _inputs(2, 20001, 9, dtype, 5, rest=rest), 2.0, dtype, up)


@pytest.mark.parametrize('rows,V,dtype', [(70000, 50, torch.float32), (40000, 200, torch.bfloat16), (9000, 3000, torch.bfloat16), (3000, 20000, torch.float16), (1100, 50000, torch.bfloat16),
                                          (600, 140000, torch.float32)])
def test_another_upstream_gradient_of_many_rows(dev, rows, V, dtype):
    """Every form of a row.  Both gradients have the same number times 1 or 3 / rows: a rounding each of the factor, the product and the result."""
    from hgq2_amd import ops

    for rest in (False, True):
        g = torch.Generator(device=dev).manual_seed(rows)
        z = (torch.randn(rows, V, generator=g, device=dev) * 4).to(dtype).requires_grad_(True)
        i, t = torch.randint(0, V, (rows, 9), generator=g, device=dev), torch.randn(rows, 9, generator=g, device=dev) * 3
        lse = torch.logsumexp(t / 2.0, 1) + 0.2 if rest else None
        (one,) = torch.autograd.grad(ops.distill_topk(z, t, i, 2.0, lse), [z])
        (three,) = torch.autograd.grad(ops.distill_topk(z, t, i, 2.0, lse) * 3.0, [z])
        one, three = one.double() * 3, three.double()
        assert ((one - three).abs() <= (HALF[dtype] + 3 * U) * (one.abs() + three.abs()) + 4 * LEAST[dtype]).all()


@pytest.mark.parametrize('rest', [False, True])
def test_the_same_index_more_than_once(dev, rest):
    z, t, i, lse, w = _inputs(5, 40, 8, torch.float32, 11, rest=rest, missing=False)
    i[0] = i[0, 0]
    i[1, 3] = i[1, 5]
    i[2, :4] = i[2, 4:]
    if rest:
        lse = torch.full((5,), 40.0)
        lse[:] = (torch.logsumexp(t.double() / 2.0, 1) + 0.1).float()
    _run(dev, (z, t, i, lse, w), 2.0, torch.float32)


# lists of teams of 8, 16, 64 and 256 threads, each of them several times as long as a team; rows that are held, read twice, and in parts
@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('rows,V,K', [(5, 40, 60), (5, 200, 60), (5, 1000, 300), (3, 5000, 700), (129, 17001, 600), (3, 50001, 900)])
def test_long_lists_with_the_same_index_more_than_once(dev, rows, V, K, rest):
    g = torch.Generator().manual_seed(V)
    z, t, i, lse, w = _inputs(rows, V, K, torch.float32, V + 1, rest=rest, weights=True)
    i[:, K // 3:K // 2] = i[:, torch.randint(0, K // 3, (K // 2 - K // 3,), generator=g)]
    i[:, -1] = i[:, 0]
    for up in (None, 3.0):
        _run(dev, (z, t, i, lse, w), 2.0, torch.float32, up)


def test_entries_without_probability(dev):
    z, t, i, _, _ = _inputs(4, 30, 6, torch.float32, 13, missing=False)
    t[0, 2:] = -math.inf
    t[1] = -math.inf  # a row without entries
    z[2, i[2, 1]] = -math.inf
    t[2, 1] = -math.inf  # 0 log 0
    _run(dev, (z, t, i, None, None), 2.0, torch.float32)
    from hgq2_amd import ops

    z[3, i[3, 0]] = -math.inf  # the teacher has what the student cannot have
    loss = ops.distill_topk(*_on(dev, z, t, i), 2.0)
    assert float(loss) == math.inf


def test_nothing_outside_the_list(dev):
    """The whole vocabulary is listed, or the rest of it masked: what rounding leaves of 1 - sum p counts as nothing."""
    z, t, i, lse, w = _inputs(6, 9, 9, torch.float32, 17, rest=True, missing=False)
    lse = (torch.logsumexp(t.double() / 2.0, 1) + 0.01).float()
    _run(dev, (z, t, i, lse, w), 2.0, torch.float32)
    z, t, i, lse, w = _inputs(6, 30, 9, torch.float32, 19, rest=True, missing=False)
    keep = torch.zeros(6, 30, dtype=torch.bool).scatter_(1, i, True)
    _run(dev, (z.masked_fill(~keep, -math.inf), t, i, lse, w), 2.0, torch.float32)
    # the list holds all but 1e-30 of the student: the rest has a maximum of its own
    z = torch.where(keep, z + 70 * 2.0, z)
    _run(dev, (z, t, i, lse, w), 2.0, torch.float32)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,V', [(5, 37), (5, 203), (5, 1003), (5, 4099), (130, 20001), (2, 20003)])
def test_a_list_at_the_end_of_the_row_that_holds_nearly_everything(dev, rows, V, dtype):
    """The row's last access reads some entries once more.  Those are of the list here: the rest (e^-140 of them) keeps a maximum of its own."""
    z, t, i, lse, w = _inputs(rows, V, 16, dtype, V, rest=True, missing=False)
    i[:] = torch.arange(V - 16, V)
    z[:, V - 16:] += 140 * 2.0
    _run(dev, (z, t, i, lse, w), 2.0, dtype)


def test_rows_that_do_not_count_may_hold_anything(dev):
    from hgq2_amd import ops

    z, t, i, lse, w = _inputs(8, 3000, 5, torch.bfloat16, 23, rest=True, weights=True)
    w[0], w[4], z[4], z[2] = 0.0, 0.0, math.nan, math.inf  # (row 2 has no entries)
    zd, td, id_, ld, wd = _on(dev, z, t, i, lse, w)
    zd.requires_grad_(True)
    loss = ops.distill_topk(zd, td, id_, 2.0, ld, wd)
    (dz,) = torch.autograd.grad(loss, [zd])
    assert math.isfinite(float(loss)) and torch.isfinite(dz).all() and not dz[[0, 2, 4]].any() and dz[1].any()
    z[1, 7] = math.nan  # and one that counts is not hidden
    loss = ops.distill_topk(z.to(dev), td, id_, 2.0, ld, wd)
    assert math.isnan(float(loss))


def test_all_missing_and_no_rows(dev):
    from hgq2_amd import ops

    for rows in (0, 3):
        z = torch.randn(rows, 12, device=dev, requires_grad=True)
        loss = ops.distill_topk(z, torch.randn(rows, 2, device=dev), torch.full((rows, 2), -1, device=dev))
        assert float(loss) == 0.0
        (dz,) = torch.autograd.grad(loss, [z])
        assert dz.shape == z.shape and not dz.any()


@pytest.mark.parametrize('pad', [1, 3, 64])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_rows_of_a_wider_buffer(dev, pad, dtype):
    from hgq2_amd import ops

    z, t, i, lse, w = _inputs(9, 1001, 12, dtype, 29, rest=True)
    buffer = torch.full((9, 1001 + pad), math.nan, dtype=dtype, device=dev)
    buffer[:, :1001] = z.to(dev)
    buffer.requires_grad_(True)
    td, id_, ld = _on(dev, t, i, lse)
    loss = ops.distill_topk(buffer[:, :1001], td, id_, 2.0, ld)
    loss.backward()
    want = _definition(z, t, i, 2.0, lse, None)
    assert abs(float(loss) - want[0]) <= want[1]
    _check(buffer.grad[:, :1001], want[2], want[3], dtype, 'dz')
    assert not buffer.grad[:, 1001:].any()
    # columns that are not next to each other, and more leading axes
    across = z.to(dev).t().contiguous().t().requires_grad_(True)
    assert abs(float(ops.distill_topk(across, td, id_, 2.0, ld)) - want[0]) <= want[1]
    cube = z.to(dev).view(3, 3, 1001).requires_grad_(True)
    got = ops.distill_topk(cube, td.view(3, 3, -1), id_.view(3, 3, -1), 2.0, ld.view(3, 3))
    assert float(got) == float(ops.distill_topk(z.to(dev), td, id_, 2.0, ld))
    (dz,) = torch.autograd.grad(got, [cube])
    _check(dz.view(9, 1001), want[2], want[3], dtype, 'dz')


def test_a_single_row_without_a_batch(dev):
    from hgq2_amd import ops

    z, t, i, _, _ = _inputs(1, 77, 4, torch.float32, 31)
    want = _definition(z, t, i, 1.0, None, None)
    assert abs(float(ops.distill_topk(*_on(dev, z[0], t[0], i[0]))) - want[0]) <= want[1]


def test_against_differences(dev):
    """(L(z + h v) - L(z - h v)) / 2 h along random v with entries below one: the third derivative of a row's loss along v is at most
    8 max|v|^3 / T times its weight over the rows (twice with the rest), so the quotient is off by 16 h^2 / (6 T), and by the losses' tolerance over h."""
    from hgq2_amd import ops

    T, h = 2.0, 2.0**-5
    for rest in (False, True):
        z, t, i, lse, w = _inputs(4, 50, 6, torch.float32, 37, T=T, rest=rest)
        zd, td, id_, ld = _on(dev, z, t, i, lse)
        (dz,) = torch.autograd.grad(ops.distill_topk(zd.requires_grad_(True), td, id_, T, ld), [zd])
        for s in range(4):
            v = torch.rand(z.shape, generator=torch.Generator().manual_seed(s)) * 2 - 1
            near = [z + k * h * v for k in (1, -1)]
            loss = [float(ops.distill_topk(k.to(dev), td, id_, T, ld)) for k in near]
            tol = sum(_definition(k, t, i, T, lse, None)[1] for k in near) / (2 * h) + 16 * h * h / (6 * T) + 50 * 4 * 64 * U
            assert abs((loss[0] - loss[1]) / (2 * h) - float((dz.double().cpu() * v.double()).sum())) <= tol


def test_kept_graphs_give_gradients_of_their_own(dev):
    from hgq2_amd import ops

    z, t, i, _, _ = _inputs(6, 200, 5, torch.float32, 41)
    zd, td, id_ = _on(dev, z, t, i)
    zd.requires_grad_(True)
    loss = ops.distill_topk(zd, td, id_)
    (a,) = torch.autograd.grad(loss, [zd], retain_graph=True)
    first = a.clone()
    a.mul_(100)
    (b,) = torch.autograd.grad(loss, [zd], torch.tensor(2.0, device=dev), retain_graph=True)
    (c,) = torch.autograd.grad(loss, [zd])
    assert torch.equal(b, 2 * first) and torch.equal(c, first)
    loss = ops.distill_topk(zd, td, id_)
    (d,) = torch.autograd.grad(loss, [zd], create_graph=True)
    with pytest.raises(RuntimeError, match='differentiable once'):
        d.sum().backward()


def test_the_same_bits_every_time_and_on_another_stream(dev):
    from hgq2_amd import ops

    for shape in ((300, 20000, 7), (3, 100000, 50), (1000, 5, 5)):
        args = _on(dev, *_inputs(*shape, torch.bfloat16, 43, rest=True, weights=True))
        z = args[0].requires_grad_(True)

        def call():
            loss = ops.distill_topk(z, args[1], args[2], 2.0, args[3], args[4])
            return loss.detach(), torch.autograd.grad(loss, [z])[0]

        want = call()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = call()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_recorded(dev):
    from hgq2_amd import ops

    for up, shape in ((1.0, (50, 3001, 6)), (3.0, (50, 3001, 6)), (1.0, (2, 40000, 6))):
        z, t, i, lse, w = _on(dev, *_inputs(*shape, torch.float32, 47, rest=True, weights=True))
        static = z.clone().requires_grad_(True)
        seed = torch.tensor(up, device=dev)

        def call():
            loss = ops.distill_topk(static, t, i, 2.0, lse, w)
            return loss.detach(), torch.autograd.grad(loss, [static], seed)[0]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loss, dz = call()
        for k in range(3):
            with torch.no_grad():
                static.copy_(z * (1 + k))
            graph.replay()
            torch.cuda.synchronize()
            got = loss.clone(), dz.clone()
            want = call()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        del loss, dz, graph


def test_recording_beside_a_living_graph_is_refused(dev):
    from hgq2_amd import ops

    z, t, i, _, _ = _on(dev, *_inputs(6, 200, 5, torch.float32, 41))
    z.requires_grad_(True)
    alive = ops.distill_topk(z, t, i)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='another stream'):
        with torch.cuda.graph(graph, stream=side):
            ops.distill_topk(z, t, i)
    assert torch.isfinite(alive)


@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('rows,V,dtype', [(130, 300_001, torch.float32), (129, 700_003, torch.bfloat16), (2, 9_000_001, torch.float16)])
def test_rows_of_many_entries(dev, rows, V, dtype, rest):
    """Sums stay within their bounds however long a row is: it is cut where a thread would add more than 64 terms.  The same definition, evaluated on the GPU."""
    from hgq2_amd import ops

    g = torch.Generator(device=dev).manual_seed(V)
    K, T = 40, 2.0
    z = (torch.randn(rows, V, generator=g, device=dev) * 4).to(dtype).requires_grad_(True)
    i = torch.stack([torch.randperm(V, generator=g, device=dev)[:K] for _ in range(rows)])
    t = torch.randn(rows, K, generator=g, device=dev) * 4 + 40
    lse = (torch.logsumexp(t.double() / T, 1) + 0.2).float() if rest else None
    loss = ops.distill_topk(z, t, i, T, lse)
    (dz,) = torch.autograd.grad(loss, [z])
    with torch.no_grad():
        assert abs(float(ops.distill_topk(z, t, i, T, lse)) - float(loss)) <= 2e-5 * abs(float(loss))
    total, tol = 0.0, 0.0
    for r in range(rows):
        zr, tr = z[r].detach().double() / T, t[r].double() / T
        log_q = zr - torch.logsumexp(zr, 0)
        q, p = log_q.exp(), (tr - (torch.logsumexp(tr, 0) if lse is None else lse[r].double())).exp()
        E = (120 + 8 * max(float(zr.max() - zr.min()), float(tr.max() - tr.min()))) * U
        gap = p.log() - log_q[i[r]]
        total, tol = total + float((p * gap).sum()), tol + E * float((p * gap.abs() + 2 * p).sum())
        share, rest_p, q_rest = torch.zeros_like(q), 0.0, 1.0
        if rest:
            rest_p = max(0.0, 1.0 - float(p.sum()))
            share = q.index_fill(0, i[r], 0.0)
            q_rest = float(share.sum())
            share /= q_rest
            total, tol = total + rest_p * math.log(rest_p / q_rest), tol + E * (abs(math.log(rest_p / q_rest)) + 2)
        at = torch.zeros_like(q).index_add_(0, i[r], p)
        P, c = float(p.sum()) + rest_p, T / rows
        want = c * (q * P - at - share * rest_p)
        bound = c * (2 * E * q * P + 2 * E * at + 2 * E * share * rest_p + E * share + 4 * U * (q + at + share))
        bound = bound + HALF[dtype] * (want.abs() + bound) + LEAST[dtype]
        assert ((dz[r].double() - want).abs() <= bound).all(), r
    assert abs(float(loss) - total * T * T / rows) <= (tol * T * T / rows) + 4 * U * abs(float(loss))
