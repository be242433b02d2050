"""What `make` builds where, by its own account (nothing is compiled)."""

import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'hgq2_amd', 'csrc')
pytestmark = pytest.mark.skipif(shutil.which('make') is None, reason='no make')


def _make(where, *args):
    return subprocess.run(['make', *args], cwd=where, capture_output=True, text=True, timeout=300)


def test_both_libraries_where_torch_is():
    got = _make(CSRC, '-n', '-B', 'all')
    assert got.returncode == 0 and '-o ../libhgq_hip.so' in got.stdout
    assert ('-o ../_host.so' in got.stdout) == (shutil.which('g++') is not None)


@pytest.mark.parametrize('missing', ['PYTHON=/nonexistent', 'CXX=/nonexistent'])
def test_the_kernels_alone_where_it_is_not(tmp_path, missing):
    """Without torch's headers or a host compiler the C ABI still builds, and the message says what was left out."""
    where = tmp_path / 'hgq2_amd' / 'csrc'
    shutil.copytree(CSRC, where, ignore=shutil.ignore_patterns('*.o'))
    shutil.copytree(os.path.join(CSRC, '..', '..', 'include'), tmp_path / 'include')
    got = _make(where, 'HIPCC=true', missing, 'all')
    assert got.returncode == 0, got.stderr[-2000:]
    assert '-o ../libhgq_hip.so' in got.stdout and '_host.so is left out' in got.stdout and '-ltorch' not in got.stdout
