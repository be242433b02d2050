"""Group normalisation: what is refused before any GPU is touched, and the layer's configuration (CPU)."""

import pytest
import torch

from hgq2_amd import _lib, ops
from hgq2_amd.host import GroupNormalization, layers


def _fwd(B=4, S=9, C=8, G=2, eps=1e-3, act=0, type=0, x=256, y=256, mean=256, rstd=256):
    """Calls that a check turns down: the addresses are never read."""
    return _lib.load().hgq_group_norm_fwd(x, None, None, y, mean, rstd, None, B, S, C, G, eps, act, type, None)


def _bwd(B=4, S=9, C=8, G=2, act=0, type=0, dy=256, x=256, mean=256, rstd=256, dx=256, dgamma=256, ws=256):
    return _lib.load().hgq_group_norm_bwd(dy, x, None, None, mean, rstd, dx, dgamma, None, ws, B, S, C, G, act, type, None)


@pytest.mark.parametrize('kw', [dict(B=-1), dict(S=-1), dict(C=0), dict(G=0), dict(G=3), dict(act=3), dict(act=-1), dict(type=3), dict(x=None),
                                dict(mean=None), dict(rstd=None), dict(B=1 << 40, S=1 << 30)])
def test_entry_points_refuse(kw):
    assert _fwd(**kw) == _lib.ERR_ARG and b'hgq_group_norm_fwd' in _lib.load().hgq_last_error()
    assert _bwd(**kw) == _lib.ERR_ARG and b'hgq_group_norm_bwd' in _lib.load().hgq_last_error()
    if not any(k in kw for k in ('act', 'x', 'mean', 'rstd')):
        shape = [kw.get(k, d) for k, d in (('B', 4), ('S', 9), ('C', 8), ('G', 2), ('type', 0))]
        assert _lib.load().hgq_group_norm_fwd_workspace(*shape) == -1 and _lib.load().hgq_group_norm_bwd_workspace(*shape) == -1


def test_entry_points_refuse_what_only_one_of_them_takes():
    assert _fwd(y=None) == _fwd(eps=-1.0) == _fwd(eps=float('nan')) == _lib.ERR_ARG
    assert _bwd(dy=None) == _bwd(ws=None) == _lib.ERR_ARG
    assert _fwd(B=1 << 31, S=1) == _lib.ERR_UNSUPPORTED
    assert _fwd(B=0, x=None) == 0 and _fwd(S=0, x=None) == 0  # nothing to do
    assert _bwd(dx=None, dgamma=None) == 0                    # nothing wanted


def test_python_refusals():
    x = torch.zeros(2, 3, 8)
    with pytest.raises(ValueError, match='GPU'):
        ops.group_norm(x, 2)
    with pytest.raises(ValueError, match='activation'):
        ops.group_norm(x, 2, activation='gelu')
    with pytest.raises(ValueError, match='negative'):
        ops.group_norm(x, 2, epsilon=-1e-3)
    with pytest.raises(ValueError, match='activation'):
        GroupNormalization(activation='tanh')
    for groups in (0, -2):
        with pytest.raises(ValueError, match='groups'):
            GroupNormalization(groups)
    with pytest.raises(ValueError, match='epsilon'):
        GroupNormalization(epsilon=-1.0)


@pytest.fixture
def cpu_build():
    from hgq2_amd.core import set_default_device

    set_default_device('cpu')
    yield
    set_default_device(None)


def test_layer_builds_as_keras_does(cpu_build):
    assert layers.GroupNormalization is GroupNormalization
    layer = GroupNormalization(4, name='norm')
    layer.build((None, 5, 5, 12))
    assert layer.gamma.shape == layer.beta.shape == (12,) and bool((layer.gamma == 1).all()) and not layer.beta.any()
    assert layer.compute_output_shape((None, 5, 5, 12)) == (None, 5, 5, 12)
    each = GroupNormalization(-1, center=False, scale=False)
    each.build((None, 7))
    assert each.groups == 7 and each.gamma is None and each.beta is None and not list(each.parameters())
    with pytest.raises(ValueError, match='groups of one size'):
        GroupNormalization(5).build((None, 4, 12))
    with pytest.raises(NotImplementedError, match='trailing'):
        GroupNormalization(2, axis=1).build((None, 4, 12))


def test_layer_is_saved_with_its_model(cpu_build, tmp_path):
    from hgq2_amd import saving
    from hgq2_amd.constraints import MinMax
    from hgq2_amd.core import Sequential
    from hgq2_amd.host import Flatten

    model = Sequential([GroupNormalization(3, epsilon=1e-5, activation='silu', gamma_constraint=MinMax(0, 2), name='norm'), Flatten(name='flat')], name='net')
    saving.build_for_shape(model, (None, 4, 6))
    with torch.no_grad():
        model.layers[0].gamma.copy_(torch.arange(6.0))
        model.layers[0].beta.copy_(-torch.arange(6.0))
    assert set(saving.variable_paths(model)) == {'net/norm/gamma', 'net/norm/beta'}
    saving.save_model(model, tmp_path / 'm.npz', input_shape=(None, 4, 6))
    other = saving.load_model(tmp_path / 'm.npz').layers[0]
    assert (other.groups, other.epsilon, other.activation, other.name) == (3, 1e-5, 'silu', 'norm')
    assert torch.equal(other.gamma, model.layers[0].gamma) and torch.equal(other.beta, model.layers[0].beta)
    assert other.gamma.constraint.bounds() == (0.0, 2.0) and other.beta.constraint is None


def test_first_use_from_several_threads():
    """Whichever thread asks first loads the host extension; the others wait for it."""
    import os
    import subprocess
    import sys

    code = '''
import threading
import torch
from hgq2_amd import _lib
_lib.load()
gate, got = threading.Barrier(8), []
def ask():
    gate.wait()
    got.append(_lib.native())
threads = [threading.Thread(target=ask) for _ in range(8)]
[t.start() for t in threads]
[t.join() for t in threads]
assert len(got) == 8 and len({id(m) for m in got}) == 1, len(got)
'''
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, '-c', code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
