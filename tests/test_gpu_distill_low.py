"""The loss against a teacher's top logits where rows lie far below zero: the same definition in 64 bits and the same tolerances.

One more term: the hardware's exponential gives zero below fp32's normal numbers, 2^-126, which D up to 133 of these rows reaches.  A gradient is c a exp(..) with
c = upstream weight T / rows and a <= P / total + p' / (sum of the rest), both of them at most one: here |c a| <= 3 * 1.5 * 0.75 * 2 < 8, so 2^-123 in all."""

import math

import pytest
import torch

from .test_gpu_distill import LEAST, _inputs, _run

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def least(monkeypatch):
    for t in (torch.float32, torch.bfloat16):
        monkeypatch.setitem(LEAST, t, 2.0**-123)


# every form of a row: teams of 8, 16, 64 (held, and read twice), 256 (held, and read twice), 512 and 1024 threads, rows in parts; lists shorter and longer than a team
FORMS = [(7, 5, 5, torch.float32), (9, 28, 3, torch.float32), (9, 56, 12, torch.bfloat16), (6, 200, 9, torch.float32), (6, 130, 40, torch.float16), (6, 1500, 50, torch.float32),
         (4100, 4000, 9, torch.bfloat16), (4, 5000, 20, torch.float32), (4, 5001, 700, torch.float16), (129, 17000, 5, torch.bfloat16), (129, 60001, 5, torch.float32),
         (129, 140001, 70, torch.float32), (1, 32000, 64, torch.bfloat16), (2, 50001, 33, torch.float32)]


@pytest.mark.parametrize('rest', [False, True])
@pytest.mark.parametrize('kind', ['low', 'lower', 'cold', 'low list', 'low stretch'])
@pytest.mark.parametrize('rows,V,K,dtype', FORMS)
def test_rows_far_below_zero(dev, rows, V, K, dtype, kind, rest):
    """A softmax does not change with a shift of its row: threads, lists, parts of a row that hold nothing add nothing, however low the others' maximum lies.  Of many rows
    eight count."""
    T = 0.01 if kind == 'cold' else 0.75
    z, t, i, lse, w = _inputs(rows, V, K, dtype, rows + V, T=T, rest=rest)
    if rows > 100:
        w = torch.zeros(rows)
        w[torch.randperm(rows, generator=torch.Generator().manual_seed(V))[:8]] = 1.5
    shift = {'low': -100 * T, 'lower': -1000 * T, 'cold': -3.0, 'low list': 0.0, 'low stretch': -100 * T}[kind]
    z = (z.float() + shift).to(dtype)
    if kind == 'low list':
        at = i.clamp(0, V - 1).long()
        z.scatter_(1, at, (z.float().gather(1, at) - 100 * T).to(dtype))
    elif kind == 'low stretch':  # threads, accesses and parts of a row that are masked as a whole
        lo, hi = (V // 3, V - V // 4) if V < 9000 else (4000, V - 9000)
        z[:, lo:hi] = -math.inf
        i = torch.where((i >= lo) & (i < hi), -1, i)
    for up in (None, 3.0):
        _run(dev, (z, t, i, lse, w), T, dtype, up)


def test_a_low_row_beside_others(dev):
    """One such row does not reach the others' mean."""
    z, t, i, lse, w = _inputs(40, 11, 4, torch.float32, 53, T=1.0, rest=True)
    z[7] -= 300.0
    _run(dev, (z, t, i, lse, w), 1.0, torch.float32)
    _run(dev, (z, t, i, None, w), 1.0, torch.float32)
