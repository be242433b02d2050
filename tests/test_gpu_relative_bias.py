"""The relative position bias: forward against the same two roundings (the sum in fp32, then to the scores' type), bit for bit; the table's
gradient against 64 bits.  There eight terms meet pairwise in fp32 (three levels, u = 2^-24 of the magnitudes each), all else is 64 bits, and the result is
rounded once: 3 u sum |terms| + 2 u |result| with the products of those errors."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24


def _buckets(T, S, n, far, both, offsets):
    """Bucket of each (sequence, query, key), each by itself from the definition."""
    m = n // 2 if both else n
    h = m // 2

    def one(d):
        k = abs(d) if both else max(-d, 0)
        b = k
        if k >= h:
            b = h
            while b + 1 < m and k**(m - h) * h**(b + 1 - h) >= far**(b + 1 - h) * h**(m - h):
                b += 1
        return b + (m if both and d > 0 else 0)

    seen = {}
    out = torch.empty(len(offsets), T, S, dtype=torch.long)
    for x, o in enumerate(offsets):
        d = torch.arange(S)[None] - torch.arange(T)[:, None] - o
        lo = int(d.min())
        line = torch.tensor([seen.setdefault(k, one(k)) for k in range(lo, int(d.max()) + 1)])
        out[x] = line[d - lo]
    return out


def _case(B, H, T, S, n, far, both, dtype, seed, offset=0):
    g = torch.Generator().manual_seed(seed)
    scores = torch.randn((B, H, T, S), generator=g).to(dtype)
    table = torch.randn((n, H), generator=g)
    dy = torch.randn((B, H, T, S), generator=g).to(dtype)
    each = offset.tolist() if isinstance(offset, torch.Tensor) else [offset] * 1
    bucket = _buckets(T, S, n, far, both, each)
    out = (scores.float() + table[bucket].permute(0, 3, 1, 2)).to(dtype)
    return scores, table, dy, bucket, out


def _grads(dy, bucket, n):
    B, H = dy.shape[:2]
    want, size = torch.zeros(n, H, dtype=torch.float64), torch.zeros(n, H, dtype=torch.float64)
    flat = bucket.expand(B, -1, -1).reshape(-1)
    for h in range(H):
        want[:, h].index_add_(0, flat, dy[:, h].double().reshape(-1))
        size[:, h].index_add_(0, flat, dy[:, h].double().abs().reshape(-1))
    return want, 3.5 * U * size + 2 * U * want.abs()


def _run(dev, B, H, T, S, n, far, both, dtype, seed, offset=0):
    from hgq2_amd import ops

    scores, table, dy, bucket, out = _case(B, H, T, S, n, far, both, dtype, seed, offset)
    s, t = scores.to(dev).requires_grad_(True), table.to(dev).requires_grad_(True)
    got = ops.relative_bias(s, t, far, both, offset.to(dev) if isinstance(offset, torch.Tensor) else offset)
    assert got.dtype == dtype and torch.equal(got.detach().cpu(), out)
    ds, dt = torch.autograd.grad(got, [s, t], dy.to(dev))
    assert torch.equal(ds.cpu(), dy)
    want, tol = _grads(dy, bucket, n)
    assert dt.dtype == torch.float32 and ((dt.double().cpu() - want).abs() <= tol).all(), float(((dt.double().cpu() - want).abs() / tol.clamp(min=1e-300)).max())


# one score; single queries and keys; odd planes; more of the batch than a run, more planes than workgroups; far distances
SHAPES = [(1, 1, 1, 1), (5000, 2, 1, 3), (1500, 3, 8, 8), (333, 2, 5, 13), (3, 2, 1, 37), (2, 3, 41, 1), (1, 1, 2, 3), (5, 3, 50, 57), (64, 4, 64, 64), (9, 2, 33, 129), (2, 1, 300, 301), (1, 2, 1, 9001), (700, 1, 3, 5), (1, 5, 517, 259)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('both', [True, False])
@pytest.mark.parametrize('shape', SHAPES)
def test_against_the_definition(dev, shape, both, dtype):
    k = sum(shape)
    _run(dev, *shape, (8, 32, 16)[k % 3], (20, 128, 60)[k % 3], both, dtype, k)


# the fewest buckets, an odd number, more than 32, 64 and 112 (other numbers of threads, and of LDS); buckets that end beyond what is looked up
@pytest.mark.parametrize('n,far,both', [(2, 2, False), (3, 9, False), (4, 3, True), (6, 5, True), (34, 100, True), (48, 30, False), (66, 200, True), (128, 500, True), (127, 9000, False),
                                        (128, 100000, True), (16, 1 << 30, False), (64, 33, False)])
def test_buckets(dev, n, far, both):
    _run(dev, 2, 2, 40, 333, n, far, both, torch.float32, n + far)
    _run(dev, 1, 1, 2, 12001, n, far, both, torch.bfloat16, n + far, offset=6000)


@pytest.mark.parametrize('offset', [-5, 7, 100, 10**12, -10**12])
def test_one_offset(dev, offset):
    _run(dev, 3, 2, 9, 30, 16, 20, True, torch.float32, 3, offset)
    _run(dev, 3, 2, 1, 30, 16, 20, False, torch.float16, 3, offset)


@pytest.mark.parametrize('kind', [torch.int32, torch.int64])
@pytest.mark.parametrize('T,S', [(1, 1000), (1, 1), (4, 133), (3, 5000)])
def test_an_offset_for_each_sequence(dev, T, S, kind):
    g = torch.Generator().manual_seed(T + S)
    for both in (True, False):
        _run(dev, 13, 3, T, S, 32, 128, both, torch.bfloat16, S, torch.randint(0, S, (13,), generator=g).to(kind))


def test_masked_scores(dev):
    from hgq2_amd import ops

    g = torch.Generator().manual_seed(5)
    scores = torch.randn((2, 3, 20, 20), generator=g).masked_fill(torch.ones(20, 20, dtype=torch.bool).triu(1), -math.inf)
    scores[1, 2, 3] = -math.inf  # a row that is masked as a whole
    scores[0, 0, 5, 2], scores[0, 0, 6, 2] = math.nan, torch.finfo(torch.float32).min
    table = torch.randn((8, 3), generator=g)
    got = ops.relative_bias(scores.to(dev), table.to(dev), 20, False).cpu()
    want = scores + table[_buckets(20, 20, 8, 20, False, [0])].permute(0, 3, 1, 2)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(1.0), want.nan_to_num(1.0))


def test_strides(dev):
    """Heads behind the batch, every other sequence, planes that are transposed or cut, no batch, a gradient that is broadcast."""
    from hgq2_amd import ops

    scores, table, dy, bucket, out = _case(6, 4, 17, 23, 16, 30, True, torch.bfloat16, 9)
    want, tol = _grads(dy, bucket, 16)
    t = table.to(dev).requires_grad_(True)
    s = scores.to(dev)
    for x in (s.transpose(0, 1).contiguous().transpose(0, 1), torch.stack([s, s], 1).reshape(12, 4, 17, 23)[::2], s.transpose(2, 3).contiguous().transpose(2, 3),
              torch.cat([s, s], 3)[..., :23], torch.cat([s, s], 2)[:, :, :17]):
        got = ops.relative_bias(x, t, 30)
        assert torch.equal(got.detach().cpu(), out)
        (dt,) = torch.autograd.grad(got, [t], dy.to(dev).transpose(0, 1).contiguous().transpose(0, 1))
        assert ((dt.double().cpu() - want).abs() <= tol).all()
    assert torch.equal(ops.relative_bias(s[0], t, 30).detach().cpu(), out[0])
    (dt,) = torch.autograd.grad(ops.relative_bias(s, t, 30).sum(), [t])  # the gradient one, broadcast
    count = torch.zeros(16, dtype=torch.float64).index_add_(0, bucket.reshape(-1), torch.ones(17 * 23, dtype=torch.float64)) * 6
    assert torch.equal(dt.double().cpu(), count[:, None].expand(16, 4))
    ts = table.to(dev).t().contiguous().t()
    assert torch.equal(ops.relative_bias(s, ts, 30).cpu(), out)


def test_far_elements_of_a_large_tensor(dev):
    """More than 2^31 elements: the last sequence is where it should be."""
    from hgq2_amd import ops

    B, H, T, S = 129, 16, 1024, 1024
    table = torch.randn(16, H, generator=torch.Generator().manual_seed(1))
    scores = torch.zeros((B, H, T, S), dtype=torch.float16, device=dev)
    with torch.no_grad():
        out = ops.relative_bias(scores, table.to(dev), 100)
    bias = table[_buckets(T, S, 16, 100, True, [0])[0]].permute(2, 0, 1).half()
    for b in (0, 127, 128):
        assert torch.equal(out[b].cpu(), bias)
    del scores
    out.zero_()
    out[128, 15, 1023, 1023] = 3.0
    out[0, 0, 0, 1023] = 2.0
    s = torch.zeros((1, 1, 1, 1), dtype=torch.float16, device=dev).expand(B, H, T, S)
    t = table.to(dev).requires_grad_(True)
    (dt,) = torch.autograd.grad(ops.relative_bias(s, t, 100), [t], out)
    want = torch.zeros(16, H)
    want[0, 15], want[15, 0] = 3.0, 2.0
    assert torch.equal(dt.cpu(), want)


def test_only_what_is_asked_for(dev):
    from hgq2_amd import ops

    s, t = torch.randn(2, 2, 5, 5, device=dev), torch.randn(4, 2, device=dev)
    with torch.no_grad():
        assert not ops.relative_bias(s, t.clone().requires_grad_(True), 9).requires_grad
    assert not ops.relative_bias(s, t, 9).requires_grad
    a = s.clone().requires_grad_(True)
    ops.relative_bias(a, t, 9).sum().backward()
    assert torch.equal(a.grad, torch.ones_like(s))
    t.requires_grad_(True)
    (d,) = torch.autograd.grad(ops.relative_bias(a, t, 9).square().sum(), [t], create_graph=True)
    with pytest.raises(RuntimeError, match='differentiable once'):
        d.sum().backward()


@pytest.mark.parametrize('shape', [(0, 2, 3, 4), (2, 0, 3, 4), (2, 2, 0, 4), (2, 2, 3, 0)])
def test_nothing_to_do(dev, shape):
    from hgq2_amd import ops

    s, t = torch.zeros(shape, device=dev, requires_grad=True), torch.randn(4, shape[1], device=dev, requires_grad=True)
    out = ops.relative_bias(s, t, 9)
    ds, dt = torch.autograd.grad(out, [s, t], torch.zeros_like(out))
    assert out.shape == shape and ds.shape == shape and dt.shape == t.shape and not dt.any()


def test_against_differences(dev):
    """The output is linear in the table, exactly so with whole numbers: a step of one in an entry moves its scores by one."""
    from hgq2_amd import ops

    g = torch.Generator().manual_seed(3)
    s = torch.randint(-50, 50, (2, 2, 21, 34), generator=g).float().to(dev)
    t = torch.randint(-50, 50, (8, 2), generator=g).float().to(dev).requires_grad_(True)
    dy = torch.randint(-8, 8, s.shape, generator=g).float().to(dev)
    (dt,) = torch.autograd.grad(ops.relative_bias(s, t, 12), [t], dy)
    for k in range(8):
        for h in range(2):
            moved = t.detach().clone()
            moved[k, h] += 1
            assert float(((ops.relative_bias(s, moved, 12) - ops.relative_bias(s, t.detach(), 12)) * dy).sum()) == float(dt[k, h])


def test_recorded_and_on_another_stream(dev):
    """Offsets, scores and table in device memory: a replay uses what they hold then.  Two recordings replayed in turn do not disturb each other."""
    from hgq2_amd import ops

    g = torch.Generator().manual_seed(11)
    feeds = [(torch.randn((3, 2, 40, 90), generator=g).to(dev), torch.randn((8, 2), generator=g).to(dev), torch.randn((3, 2, 40, 90), generator=g).to(dev),
              torch.randint(0, 50, (3,), generator=g).to(dev)) for _ in range(3)]

    def both(s, t, dy, o):
        out = ops.relative_bias(s, t, 30, False, o)
        return (out.detach(), *torch.autograd.grad(out, [s, t], dy))

    leaf = lambda x: x.clone().requires_grad_(True)  # noqa: E731
    eager = [both(leaf(s), leaf(t), dy, o) for s, t, dy, o in feeds]
    side, recorded = torch.cuda.Stream(), []
    for _ in range(2):
        mine = [leaf(feeds[0][0]), leaf(feeds[0][1]), feeds[0][2].clone(), feeds[0][3].clone()]
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
        both(leaf(feeds[2][0]), leaf(feeds[2][1]), *feeds[2][2:])
        torch.cuda.synchronize()
        for _, _, out in recorded:
            assert all(torch.equal(a, b) for a, b in zip(out, eager[k])), k


def test_recording_beside_a_living_graph_is_refused(dev):
    from hgq2_amd import ops

    s, t = torch.randn(2, 2, 5, 5, device=dev), torch.nn.Parameter(torch.randn(4, 2, device=dev))
    living = ops.relative_bias(s, t, 9)
    side = torch.cuda.Stream()
    with pytest.raises(RuntimeError, match='table belongs to a graph of another stream'):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            ops.relative_bias(s, t, 9)
    del living


def test_an_offset_for_each_of_no_sequences_and_none_for_some(dev):
    from hgq2_amd import ops

    table = torch.randn(8, 2, device=dev)
    none = torch.empty(0, dtype=torch.long, device=dev)
    assert ops.relative_bias(torch.empty(0, 2, 3, 4, device=dev), table, 9, offset=none).shape == (0, 2, 3, 4)
    with pytest.raises(ValueError, match='offset must be'):
        ops.relative_bias(torch.zeros(32, 2, 1, 4, device=dev), table, 9, offset=none)


@pytest.mark.parametrize('first', [[1, 2, 5 - 2**32], [1 - 2**32, 2, 5], [1, 2, 5 + 2**32], [1, 2, -5]])
def test_first_distances_of_the_operators_that_are_none(dev, first):
    from hgq2_amd import _lib

    s, t = torch.zeros(1, 2, 3, 4, device=dev), torch.zeros(8, 2, device=dev)
    with pytest.raises(_lib.HGQLibraryError, match='first distances'):
        torch.ops.hgq.relative_bias_fwd(s, t, None, 0, first, True)
    with pytest.raises(_lib.HGQLibraryError, match='first distances'):
        torch.ops.hgq.relative_bias_bwd(s, None, 0, first, True)


def test_a_table_of_more_elements_than_a_launch_has_wavefronts(dev):
    """2^19 + 9 heads of one score each and 128 buckets: the score's bucket takes its gradient, all else is zero."""
    from hgq2_amd import ops

    heads = (1 << 19) + 9
    scores, table = torch.zeros(1, heads, 1, 1, device=dev), torch.zeros(128, heads, device=dev, requires_grad=True)
    dy = torch.randn(1, heads, 1, 1, device=dev)
    (dt,) = torch.autograd.grad(ops.relative_bias(scores, table, 128, True, offset=-3), [table], dy)
    assert torch.equal(dt[64 + 3], dy.view(-1))  # (three ahead: the fourth bucket of that half)
    dt[64 + 3] = 0
    assert not dt.any()
