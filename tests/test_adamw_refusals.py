"""AdamW and the global gradient norm: descriptor layouts against the C compiler's, and the calls that are refused before any
GPU is touched."""

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from hgq2_amd import _lib, ops
from hgq2_amd.train import AdamW, train_step_for

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which('g++') is None, reason='no host compiler')
def test_layouts_match_the_header(tmp_path):
    lines = ['#include <cstddef>', '#include <cstdio>', f'#include "{ROOT}/include/hgq_hip.h"', 'int main() {']
    want = []
    for name, cls in (('hgq_adamw_item', ops._AdamwItem), ('hgq_adamw_state', ops._AdamwState)):
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        want.append(f'{name} {ctypes.sizeof(cls)}')
        for field, *_ in cls._fields_:
            lines.append(f'printf("{name}.{field} %zu %zu\\n", offsetof({name}, {field}), sizeof((({name} *)0)->{field}));')
            d = getattr(cls, field)
            want.append(f'{name}.{field} {d.offset} {d.size}')
    for name, value in (('HGQ_ADAMW_BLOCK', ops.ADAMW_BLOCK), ('HGQ_ADAMW_TICKETS', ops.ADAMW_TICKETS), ('HGQ_TYPE_F32', 0), ('HGQ_TYPE_BF16', 1), ('HGQ_TYPE_F16', 2)):
        lines.append(f'printf("{name} %ld\\n", (long)({name}));')
        want.append(f'{name} {value}')
    (tmp_path / 'layout.cpp').write_text('\n'.join(lines + ['return 0;', '}']))
    subprocess.run(['g++', '-o', str(tmp_path / 'layout'), str(tmp_path / 'layout.cpp')], check=True)
    assert subprocess.run([str(tmp_path / 'layout')], check=True, capture_output=True, text=True).stdout.split('\n')[:-1] == want


def test_descriptor_words():
    """The words that the Python side writes are the fields of the structure."""
    from array import array

    words = array('q', (1, 2, 3, 4, 5, 6, 7, 8, *ops._adamw_limits_words(0.5, -2.0, float('inf'), 0.25), 2, 11, 12, 13, 14, 21, 22, 23, 24))
    assert len(words) == ops._ADAMW_WORDS and ctypes.sizeof(ops._AdamwItem) == 8 * ops._ADAMW_WORDS
    it = ops._AdamwItem.from_buffer_copy(words.tobytes())
    assert [it.w, it.g, it.m, it.v, it.m_scale, it.v_scale, it.n, it.first] == [1, 2, 3, 4, 5, 6, 7, 8]
    assert (it.l1, it.lo, it.hi, it.decay, it.type) == (0.5, -2.0, float('inf'), 0.25, 2)
    assert list(it.side) == [11, 12, 13, 14] and list(it.side_scale) == [21, 22, 23, 24]
    st = ops._AdamwState.from_buffer_copy(ops.adamw_state('cpu', 0.125, 3, 0.5, 0.25).numpy().tobytes())
    assert (st.step, st.beta_1_power, st.beta_2_power, st.lr) == (3, 0.125, 0.015625, 0.125) and not any(any(t) for t in st.ticket)


def _item(**kw):
    it = ops._AdamwItem(w=256, g=256, m=256, v=256, m_scale=256, v_scale=256, n=16, first=0, lo=float('-inf'), hi=float('inf'))
    for k, v in kw.items():
        setattr(it, k, v)
    return it


def _update(it, bits=32, b1=0.9, b2=0.999, eps=1e-7, clip=0.0, parts=None, n_parts=0, state=256, count=1, terms=None, n_terms=0, out=None):
    """Calls that a check turns down: the addresses are never read."""
    return _lib.load().hgq_adamw_update_multi(ctypes.byref(it) if it is not None else None, count, bits, state, b1, b2, eps, clip, parts, n_parts,
                                              None, 0, terms, n_terms, out, None)


@pytest.mark.parametrize('item,kw', [
    (dict(w=None), {}), (dict(g=None), {}), (dict(m=None), {}), (dict(v=None), {}), (dict(n=-1), {}), (dict(n=(1 << 40) + 1), {}),
    (dict(type=3), {}), (dict(type=-1), {}), (dict(m_scale=None), dict(bits=8)), (dict(v_scale=None), dict(bits=8)), (dict(first=4), dict(bits=8)),
    (dict(first=-256), dict(bits=8)), ({}, dict(bits=16)), ({}, dict(state=None)), ({}, dict(count=-1)), ({}, dict(b1=1.0)), ({}, dict(b2=-0.1)),
    ({}, dict(b1=float('nan'))), ({}, dict(eps=-1e-7)), ({}, dict(n_parts=4, parts=256)), ({}, dict(n_parts=4, clip=1.0)), ({}, dict(n_parts=-1)),
    ({}, dict(n_terms=1)), ({}, dict(n_terms=65, terms=256, out=256)),
])
def test_the_update_refuses(item, kw):
    assert _update(_item(**item), **kw) == _lib.ERR_ARG
    assert b'hgq_adamw_update_multi' in _lib.load().hgq_last_error()


def test_null_items_are_refused():
    assert _update(None) == _lib.ERR_ARG
    lib = _lib.load()
    assert lib.hgq_global_norm(None, 1, None, None, None) == _lib.ERR_ARG and lib.hgq_global_norm_parts(None, 1) == -1
    it = _item(g=None)
    assert lib.hgq_global_norm(ctypes.byref(it), 1, 256, 256, None) == _lib.ERR_ARG
    it = _item(w=None, m=None, v=None)  # the norm reads the gradient alone
    assert lib.hgq_global_norm_parts(ctypes.byref(it), 1) == 1
    assert lib.hgq_global_norm(ctypes.byref(it), 1, None, 256, None) == _lib.ERR_ARG  # no workspace


def test_python_refusals():
    p = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match='GPU'):
        AdamW([p])
    with pytest.raises(ValueError, match='at least one'):
        AdamW([torch.nn.Parameter(torch.zeros(4), requires_grad=False)])
    for kw in (dict(state_bits=4), dict(beta_1=1.0), dict(beta_2=-0.5), dict(epsilon=-1.0), dict(weight_decay=-0.1), dict(global_clipnorm=0.0),
               dict(global_clipnorm=-1.0)):
        with pytest.raises(ValueError, match='bits|expected|positive'):
            AdamW([p], **kw)
    with pytest.raises(ValueError, match='GPU'):
        ops.global_norm([p])
    with pytest.raises(ValueError, match='at least one'):
        ops.global_norm([None])
    state, moments = ops.adamw_state('cpu', 0.1), ops.adamw_moments(4, 'cpu')
    with pytest.raises(ValueError, match='GPU'):
        ops.adamw_update_multi_([p], [torch.zeros(4)], [moments], state)
    with pytest.raises(ValueError, match='length'):
        ops.adamw_update_multi_([p], [torch.zeros(4)], [], state)
    with pytest.raises(ValueError, match='positive'):
        ops.adamw_update_multi_([p], [torch.zeros(4)], [moments], state, clipnorm=0.0)
    with pytest.raises(ValueError, match='bits'):
        ops.adamw_moments(4, 'cpu', 16)


def test_unknown_optimizers_are_refused():
    with pytest.raises(ValueError, match='optimizer'):
        train_step_for(None, None, None, optimizer='lion')
    with pytest.raises(ValueError, match='SGD only'):
        train_step_for(None, None, None, optimizer='adamw', fused=True)


def test_moments_before_the_first_step():
    m, v = ops.adamw_moments(300, 'cpu')
    assert m.dtype == v.dtype == torch.float32 and m.numel() == v.numel() == 300 and not m.any() and not v.any()
    for t, (dtype, n) in zip(ops.adamw_moments(300, 'cpu', 8), ((torch.float8_e4m3fn, 300), (torch.float8_e8m0fnu, 2)) * 2):
        assert t.dtype == dtype and t.numel() == n


def test_missing_host_extension_fails_loudly(monkeypatch):
    monkeypatch.setattr(_lib, '_native', None)
    monkeypatch.setattr(_lib, '_HERE', '/nonexistent')
    with pytest.raises(_lib.HGQLibraryError, match='not built'):
        _lib.native()


def test_operators_without_data():
    """Shapes and types on fake tensors, as tracing sees the operators; CPU tensors reach the check that refuses them."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    _lib.native()
    with FakeTensorMode():
        x, c = torch.empty(2, 5, 8, dtype=torch.bfloat16, device='cuda'), torch.empty(8, device='cuda')
        y, stats = torch.ops.hgq.group_norm_fwd(x, c, c, 4, 1e-3, 0)
        assert y.shape == x.shape and y.dtype == x.dtype and stats.shape == (2, 2, 4) and stats.dtype == torch.float64
        dx, dg, db = torch.ops.hgq.group_norm_bwd(y, x, c, c, stats, 4, 0, True, True, False)
        assert dx.shape == x.shape and dg.shape == (8,) and db.numel() == 0
        assert torch.ops.hgq.global_norm([x, c]).shape == ()
        out = ops.group_norm(x, 4, c, c, activation='silu')
        assert out.shape == x.shape and ops.global_norm([x]).dtype == torch.float32
    z = torch.zeros(2, 5, 8)
    with pytest.raises(ValueError, match='GPU'):
        torch.ops.hgq.group_norm_fwd(z, z[0, 0], z[0, 0], 4, 1e-3, 0)
    with pytest.raises(TypeError, match='tensor'):
        ops.group_norm(3.0, 4)


def test_an_epsilon_that_is_no_normal_number_and_memory_that_is_shared():
    p = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match='2\\^-126'):
        AdamW([p], epsilon=1e-40)
    assert _update(_item(), eps=1e-40) == _lib.ERR_ARG
    buf = torch.zeros(10)
    ops._need_apart('variables', [buf[5:], buf[:5], buf[3:3]])
    with pytest.raises(ValueError, match='variables share memory'):
        ops._need_apart('variables', [buf[4:], buf[:5]])
    with pytest.raises(ValueError, match='variables share memory'):
        ops._need_apart('variables', [buf[2:3], buf[:5]])
