"""Operators are there as soon as the package is imported, whichever of them is asked for first (each in a process of its own)."""

import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(code):
    done = subprocess.run([sys.executable, '-c', code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_by_name_after_the_import():
    _run('''
import torch, hgq2_amd
from hgq2_amd import _lib
for name in ('group_norm_fwd', 'group_norm_bwd', 'global_norm', 'adamw_update_multi', 'quantize_fwd'):
    getattr(torch.ops.hgq, name)
assert _lib._lib is None  # (the HIP library is loaded by the first call, which settles what the environment says then)
from torch._subclasses.fake_tensor import FakeTensorMode
with FakeTensorMode():
    x = torch.empty(2, 5, 8, device='cuda')
    assert torch.ops.hgq.global_norm([x]).shape == ()
z = torch.zeros(2, 5, 8)
try:
    torch.ops.hgq.group_norm_fwd(z, z[0, 0], z[0, 0], 4, 1e-3, 0)
except ValueError as e:
    assert 'GPU' in str(e)
else:
    raise SystemExit('not refused')
''')


def test_a_missing_extension_does_not_stop_the_import():
    _run('''
import os
exists = os.path.exists
os.path.exists = lambda p: not str(p).endswith('_host.so') and exists(p)
from hgq2_amd import _lib, ops
import torch
try:
    ops.global_norm([torch.zeros(3)])
except _lib.HGQLibraryError as e:
    assert 'not built' in str(e)
else:
    raise SystemExit('not refused')
''')


@pytest.mark.gpu
def test_the_first_call_of_all_by_name(dev):
    _run('''
import torch, hgq2_amd
x = torch.full((3, 4), 2.0, device='cuda')
assert float(torch.ops.hgq.global_norm([x])) == 48 ** 0.5 or abs(float(torch.ops.hgq.global_norm([x])) - 48 ** 0.5) < 1e-6
y, stats = torch.ops.hgq.group_norm_fwd(x.view(1, 3, 4), torch.ones(4, device='cuda'), torch.zeros(4, device='cuda'), 2, 1e-3, 0)
assert not y.any() and stats.shape == (2, 1, 2)
''')
