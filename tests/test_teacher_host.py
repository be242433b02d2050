"""Distillation, relative position bias and the norms around a residual sum: what is refused before any GPU is touched (CPU)."""

import ctypes
import math

import pytest
import torch

from hgq2_amd import _lib, ops


def _refused(rc, name, code=None):
    assert rc == (_lib.ERR_ARG if code is None else code) and name in _lib.load().hgq_last_error(), rc


def _distill(fwd=True, z=256, z_stride=9, t=256, t_type=0, index=256, index_bytes=4, loss=256, ws=256, up=256, stats=256, dz=256, rows=3, V=9, K=2, T=1.0, type=0):
    """Calls that a check turns down: the addresses are never read."""
    lib = _lib.load()
    if fwd:
        return lib.hgq_distill_topk_fwd(z, z_stride, t, t_type, index, index_bytes, None, None, loss, None, None, ws, rows, V, K, T, type, None)
    return lib.hgq_distill_topk_bwd(z, z_stride, t, t_type, index, index_bytes, None, None, up, stats, dz, 0, rows, V, K, T, type, None)


@pytest.mark.parametrize('kw', [dict(rows=-1), dict(V=0), dict(K=0), dict(T=0.0), dict(T=-1.0), dict(T=math.nan), dict(T=math.inf), dict(T=1e-31), dict(T=1e31), dict(type=3), dict(t_type=-1), dict(index_bytes=2),
                                dict(z=None), dict(t=None), dict(index=None), dict(z_stride=-9)])
def test_distillation_entry_points(kw):
    _refused(_distill(**kw), b'hgq_distill_topk_fwd')
    _refused(_distill(fwd=False, **kw), b'hgq_distill_topk_bwd')


def test_distillation_limits():
    _refused(_distill(loss=None), b'null')
    _refused(_distill(ws=None), b'null')
    for k in ('up', 'stats', 'dz'):
        _refused(_distill(fwd=False, **{k: None}), b'null')
    for kw in (dict(K=1025), dict(K=65, V=7), dict(V=(1 << 30) + 1), dict(rows=1 << 41)):
        _refused(_distill(**kw), b'hgq_distill_topk_fwd', _lib.ERR_UNSUPPORTED)
        _refused(_distill(fwd=False, **kw), b'hgq_distill_topk_bwd', _lib.ERR_UNSUPPORTED)
        assert _lib.load().hgq_distill_topk_workspace(kw.get('rows', 3), kw.get('V', 9), kw.get('K', 2), 0) == -1
    assert _distill(fwd=False, rows=0, z=None) == 0


@pytest.mark.parametrize('rows,V,K', [(1, 5, 5), (16384, 5, 5), (7, 64, 65), (1, 32000, 64), (300, 32000, 64), (2, 300000, 1000), (4096, 131072, 100), (4096, 1 << 20, 100)])
def test_distillation_workspace(rows, V, K):
    """A sum for each workgroup, and two numbers for each part of a row where rows are cut: never more than a small part of the logits."""
    for rest in (0, 1):
        n = _lib.load().hgq_distill_topk_workspace(rows, V, K, rest)
        assert 2 <= n <= 2 * rows + max(2 * rows * V // 4096, 0) + 2 * rows


def _bias(fwd=True, x=256, table=256, out=256, ws=256, B=2, H=2, T=3, S=4, first=(1, 2, 5), m=None, both=1, offset_bytes=8, type=0):
    lib, n = _lib.load(), len(first) + 1 if m is None else m
    first = (ctypes.c_int * max(1, len(first)))(*first) if first is not None else None
    if fwd:
        return lib.hgq_relative_bias_fwd(x, 24, 12, table, out, B, H, T, S, first, n, both, 0, None, offset_bytes, type, None)
    return lib.hgq_relative_bias_bwd(x, 24, 12, table, ws, B, H, T, S, first, n, both, 0, None, offset_bytes, type, None)


@pytest.mark.parametrize('kw', [dict(B=-1), dict(H=-1), dict(T=-1), dict(S=-1), dict(type=3), dict(offset_bytes=2), dict(first=(0, 2)), dict(first=(3, 2)), dict(first=(1, (1 << 30) + 1)),
                                dict(first=(), m=1), dict(x=None), dict(table=None)])
def test_bias_entry_points(kw):
    _refused(_bias(**kw), b'hgq_relative_bias_fwd')
    _refused(_bias(fwd=False, **kw), b'hgq_relative_bias_bwd')


def test_bias_limits():
    for kw in (dict(first=tuple(range(1, 65))), dict(first=tuple(range(1, 129)), both=0), dict(T=1 << 16, S=1 << 16), dict(B=(1 << 30) + 1), dict(H=1 << 21)):
        _refused(_bias(**kw), b'hgq_relative_bias_fwd', _lib.ERR_UNSUPPORTED)
        _refused(_bias(fwd=False, **kw), b'hgq_relative_bias_bwd', _lib.ERR_UNSUPPORTED)
    _refused(_bias(out=None), b'null')
    _refused(_bias(fwd=False, ws=None), b'null')
    assert _bias(B=0, x=None) == _bias(S=0, x=None) == _bias(fwd=False, H=0, x=None) == 0
    assert _lib.load().hgq_relative_bias_bwd_workspace(2, 2, 3, 4, 65, 1) == _lib.load().hgq_relative_bias_bwd_workspace(2, 2, -3, 4, 4, 1) == -1


def _residual(fwd=True, x=256, u=256, gate=None, y=256, h=256, dy=256, dh=256, r_u=256, r_y=256, ws=256, rows=6, P=1, C=8, scale=1.0, eps=1e-6, act=0, type=0, du=256, dgate=None, dpost=256):
    lib = _lib.load()
    if fwd:
        return lib.hgq_residual_norm_fwd(x, u, gate, None, None, y, h, r_u, r_y, rows, P, C, scale, eps, act, type, None)
    return lib.hgq_residual_norm_bwd(dy, dh, x, u, gate, None, None, r_u, r_y, 256, du, dgate, dpost, 256, ws, rows, P, C, scale, eps, act, type, None)


@pytest.mark.parametrize('kw', [dict(rows=-1), dict(P=0), dict(P=4), dict(C=0), dict(eps=-1.0), dict(eps=math.nan), dict(scale=math.nan), dict(act=2), dict(act=-1), dict(type=3), dict(x=None),
                                dict(u=None, gate=256)])
def test_residual_entry_points(kw):
    _refused(_residual(**kw), b'hgq_residual_norm_fwd')
    _refused(_residual(fwd=False, **kw), b'hgq_residual_norm_bwd')


def test_residual_limits():
    for kw in (dict(h=None), dict(y=None)):
        _refused(_residual(**kw), b'null')
    for kw in (dict(r_u=None), dict(r_y=None), dict(dy=None, dh=None), dict(ws=None), dict(dgate=256), dict(u=None), dict(u=None, du=None)):
        _refused(_residual(fwd=False, **kw), b'null')
    for kw in (dict(C=(1 << 28) + 1), dict(rows=1 << 41)):
        _refused(_residual(**kw), b'hgq_residual_norm_fwd', _lib.ERR_UNSUPPORTED)
        _refused(_residual(fwd=False, **kw), b'hgq_residual_norm_bwd', _lib.ERR_UNSUPPORTED)
    assert _residual(rows=0, x=None) == 0
    assert _lib.load().hgq_residual_norm_bwd_workspace(6, 4, 8, 0) == -1 and _lib.load().hgq_residual_norm_bwd_workspace(0, 1, 8, 0) == 0


def test_python_refusals():
    z, i = torch.zeros(3, 7), torch.zeros(3, 2, dtype=torch.long)
    with pytest.raises(ValueError, match='GPU'):
        ops.distill_topk(z, z[:, :2], i)
    with pytest.raises(ValueError, match='leading axes'):
        ops.distill_topk(z, z[:2, :2], i)
    with pytest.raises(ValueError, match='teacher_indices'):
        ops.distill_topk(z, z[:, :2], i[:, :1])
    with pytest.raises(ValueError, match='teacher_lse'):
        ops.distill_topk(z, z[:, :2], i, teacher_lse=z)
    with pytest.raises(ValueError, match='sample_weight'):
        ops.distill_topk(z, z[:, :2], i, sample_weight=z[:2, 0])
    with pytest.raises(ValueError, match='detach'):
        ops.distill_topk(z, z[:, :2].clone().requires_grad_(True), i)
    with pytest.raises(TypeError, match='tensor'):
        ops.distill_topk(3.0, z, i)

    s, t = torch.zeros(1, 2, 3, 4), torch.zeros(4, 2)
    with pytest.raises(ValueError, match='GPU'):
        ops.relative_bias(s, t, 9)
    with pytest.raises(ValueError, match='scores'):
        ops.relative_bias(s[0, 0], t, 9)
    with pytest.raises(ValueError, match='buckets, heads'):
        ops.relative_bias(s, t[0], 9)
    with pytest.raises(ValueError, match='even'):
        ops.relative_bias(s, t[:3], 9)
    with pytest.raises(ValueError, match='at most 128'):
        ops.relative_bias(s, torch.zeros(130, 2))
    with pytest.raises(ValueError, match='max_distance'):
        ops.relative_bias(s, torch.zeros(32, 2), 8)
    with pytest.raises(ValueError, match='max_distance'):
        ops.relative_bias(s, t, (1 << 30) + 1)
    with pytest.raises(ValueError, match='two buckets'):
        ops.relative_bias(s, t[:2], 9)
    with pytest.raises(TypeError):
        ops.relative_bias(s, t, 9, offset=2.5)  # (a position is a whole number)

    x = torch.zeros(2, 3, 8)
    with pytest.raises(ValueError, match='GPU'):
        ops.residual_norm(x, x)
    with pytest.raises(ValueError, match='GPU'):
        ops.rms_norm(x)
    with pytest.raises(ValueError, match='gate_activation'):
        ops.residual_norm(x, x, gate=x, gate_activation='tanh')
    with pytest.raises(ValueError, match='negative'):
        ops.rms_norm(x, epsilon=-1.0)
    with pytest.raises(ValueError, match='update'):
        ops.residual_norm(x, x[0])
    with pytest.raises(ValueError, match='update'):
        ops.residual_norm(x, None)
    with pytest.raises(ValueError, match='post_gamma'):
        ops.residual_norm(x, x, post_gamma=x[0, 0, :3])
    for gate in (x[0], x[:1, 0], x[:, :2], x[..., :4]):
        with pytest.raises(ValueError, match='gate'):
            ops.residual_norm(x, x, gate=gate)


@pytest.mark.parametrize('offset', [torch.empty(0, dtype=torch.long), torch.zeros(2, dtype=torch.long), torch.zeros(4, dtype=torch.int32), torch.zeros((), dtype=torch.long),
                                    torch.zeros(3, 1, dtype=torch.long), torch.zeros(6, dtype=torch.long)[::2], torch.zeros(3), torch.zeros(3, dtype=torch.int16)])
def test_offsets_that_are_not_one_for_each_sequence(offset):
    with pytest.raises(ValueError, match='offset must be'):
        ops.relative_bias(torch.zeros(3, 2, 3, 4), torch.zeros(4, 2), 9, offset=offset)
    with pytest.raises(ValueError, match='offset must be'):
        ops.relative_bias(torch.zeros(2, 3, 4), torch.zeros(4, 2), 9, offset=offset)
    with pytest.raises(ValueError, match='GPU'):  # (one that is)
        ops.relative_bias(torch.zeros(3, 2, 3, 4), torch.zeros(4, 2), 9, offset=torch.zeros(3, dtype=torch.long))


def test_batches_of_several_targets():
    from hgq2_amd.train import _copy_batch, _each

    example = (torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.long), None)
    to = _each(torch.Tensor.clone, example)
    batch = (torch.rand(2, 3), torch.randint(0, 9, (2, 3)), None)
    _copy_batch(to, list(batch))
    assert torch.equal(to[0], batch[0]) and torch.equal(to[1], batch[1]) and to[2] is None and not example[0].any()
    _copy_batch(None, None)
    kept = _each(torch.Tensor.clone, to)
    for wrong in (batch[:2], (*batch[:2], torch.rand(2)), (batch[0], None, None), (batch[0][:, :1], *batch[1:]), (batch[0], batch[1][:1], None), torch.rand(3, 2, 3), None):
        with pytest.raises(ValueError, match='targets'):
            _copy_batch(to, wrong)
    with pytest.raises(ValueError, match='targets'):
        _copy_batch(None, batch)
    assert torch.equal(to[0], kept[0]) and torch.equal(to[1], kept[1])
    single = torch.zeros(4)
    _copy_batch(single, torch.arange(4.0))
    assert torch.equal(single, torch.arange(4.0))


@pytest.mark.parametrize('n,far', [(2, 2), (2, 100), (3, 9), (8, 40), (16, 128), (32, 128), (32, 33), (64, 500), (20, 1 << 30)])
def test_first_distances(n, far):
    """The definition bucket by bucket, in whole numbers: the bucket of a distance is how many first distances are not above it."""
    first, h = ops.relative_buckets(n, far), n // 2
    assert len(first) == n - 1 and list(first) == sorted(first) and first[-1] <= far and list(first[:h]) == list(range(1, h + 1))
    for b, f in enumerate(first[h:], h + 1):
        reached = lambda k: k**(n - h) * h**(b - h) >= far**(b - h) * h**(n - h)  # noqa: E731
        assert reached(f) and not reached(f - 1)


def test_registered_for_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        z, i = torch.empty(3, 9, device='cuda'), torch.empty(3, 2, dtype=torch.long, device='cuda')
        none = torch.empty(0, device='cuda')
        loss, stats, dz = torch.ops.hgq.distill_topk_fwd(z, z[:, :2], i, none, None, 1.0)
        assert loss.shape == () and stats.shape == (3, 4) and dz.shape == z.shape
        assert torch.ops.hgq.distill_topk_bwd(loss, z, z[:, :2], i, none, None, stats, 1.0).shape == z.shape
        assert torch.ops.hgq.distill_topk_loss(z, z[:, :2], i, None, None, 1.0).shape == ()
        s, t = torch.empty(2, 4, 5, 6, device='cuda'), torch.empty(8, 4, device='cuda')
        assert torch.ops.hgq.relative_bias_fwd(s, t, none, 0, [1, 2, 5], True).shape == s.shape
        assert torch.ops.hgq.relative_bias_bwd(s, None, 0, [1, 2, 5], True).shape == t.shape
        x = torch.empty(2, 3, 8, device='cuda')
        y, h, r = torch.ops.hgq.residual_norm_fwd(x, x, none, None, None, 1, 1.0, 1e-6, 0)
        assert y.shape == h.shape == x.shape and r.shape == (12,)
        assert [t.shape for t in torch.ops.hgq.residual_norm_values(x, x, None, None, none, 1, 1.0, 1e-6, 0)] == [x.shape] * 2
        assert [t.shape for t in torch.ops.hgq.residual_norm_values(x, None, None, None, None, 1, 1.0, 1e-6, 0)] == [x.shape]
        got = torch.ops.hgq.residual_norm_bwd(x, None, x, x, none, none, None, r, 1, 1.0, 1e-6, 0, True, True, False, True, False)
        assert [tuple(g.shape) for g in got] == [(2, 3, 8), (2, 3, 8), (0,), (8,), (0,)]


@pytest.fixture
def cpu_build():
    from hgq2_amd.core import set_default_device

    set_default_device('cpu')
    yield
    set_default_device(None)


def test_layers_refuse_what_cannot_be():
    from hgq2_amd.host import Flatten, ResidualBlocks, RMSNormalization
    from hgq2_amd.layers import QMultiHeadAttention

    with pytest.raises(ValueError, match='at least one'):
        ResidualBlocks([])
    with pytest.raises(ValueError, match='as many gates'):
        ResidualBlocks([Flatten()], [None, None])
    with pytest.raises(ValueError, match='gate_activation'):
        ResidualBlocks([Flatten()], gate_activation='relu')
    for make in (lambda: ResidualBlocks([Flatten()], epsilon=-1.0), lambda: RMSNormalization(epsilon=math.nan)):
        with pytest.raises(ValueError, match='epsilon'):
            make()
    with pytest.raises(NotImplementedError, match='trailing'):
        RMSNormalization(axis=1).build((2, 3, 4))
    for kw in (dict(relative_buckets=7), dict(relative_buckets=130), dict(relative_buckets=-2)):
        with pytest.raises(ValueError, match='relative_buckets'):
            QMultiHeadAttention(2, 8, **kw)
    with pytest.raises(ValueError, match='max_distance'):
        QMultiHeadAttention(2, 8, relative_buckets=32, relative_max_distance=8)
    with pytest.raises(ValueError, match="'distill_topk'"):
        from hgq2_amd.train import train_step_for

        train_step_for(None, None, None, loss='kl')


def test_layers_configurations_and_variables(cpu_build):
    from hgq2_amd.host import ResidualBlocks, RMSNormalization, layers
    from hgq2_amd.layers import QDense, QMultiHeadAttention
    from hgq2_amd.saving import build_for_shape, deserialize, serialize, variable_paths

    assert layers.RMSNormalization is RMSNormalization
    layer = ResidualBlocks([QMultiHeadAttention(2, 8, relative_buckets=9, relative_max_distance=30, relative_bidirectional=False, name='attention'), QDense(16, name='dense')],
                           [None, QDense(16, name='gate')], scale=0.25, name='blocks')
    again = deserialize(serialize(layer))
    for made in (layer, again):
        build_for_shape(made, (None, 5, 16))
    paths = variable_paths(layer)
    assert list(paths) == list(variable_paths(again)) and [tuple(t.shape) for t in paths.values()] == [tuple(t.shape) for t in variable_paths(again).values()]
    assert tuple(paths['blocks/attention/relative_bias'].shape) == (9, 2) and {f'blocks/{n}' for n in ('gamma_0', 'gamma_1', 'gamma_2', 'post_0', 'post_1', 'gate/kernel')} <= set(paths)
    assert again._gated == [False, True] and again.scale == 0.25 and again.blocks[0]._relative == (9, 30, False)
    assert 'relative_buckets' not in QMultiHeadAttention(2, 8).get_config()
