"""Roundings of the AdamW step, where a value lies on a border and one unit in the last place shows."""

import numpy as np
import pytest
import torch

from .test_gpu_adamw import BLOCK, _philox, _values

pytestmark = pytest.mark.gpu


def test_the_root_is_rounded(dev):
    """With beta_2 = 0 the second moment is g g, rounded, and the rounded root of that is |g| again (in a binary format, away from its
    ends).  Gradients are laid exactly on the borders of the stochastic rounding - a whole number of steps less the random number that is
    added - so the code is the upper one for |g| itself and the lower one for anything below it."""
    from hgq2_amd import ops

    n, seed = 1 << 20, 77
    gen = torch.Generator().manual_seed(22)
    h = torch.from_numpy((_philox(np.arange(n // 4, dtype=np.uint64), 1, seed) >> np.uint64(16)).astype(np.int64)).double()
    k = torch.randint(8, 16, (n,), generator=gen).double()
    steps = torch.where(h > 0, k + 1 - h / 65536, k)  # 20 bits
    want = torch.where(h > 0, k + 1, k)
    steps[::BLOCK] = want[::BLOCK] = 15.0  # (every block's largest magnitude lies in [128, 256) of its scale)
    exponent = torch.arange(n // BLOCK) % 113 - 62  # of scales: g g stays a normal number
    scale = torch.pow(2.0, exponent.double()).repeat_interleave(BLOCK)
    g64 = steps * 16 * scale
    g = g64.float()
    assert torch.equal(g.double(), g64)
    h[::BLOCK] = 0
    w, moments = torch.zeros(n, device=dev), ops.adamw_moments(n, dev, 8)
    ops.adamw_update_multi_([w], [(g * torch.where(torch.rand(n, generator=gen) < 0.5, -1.0, 1.0)).to(dev)], [moments], ops.adamw_state(dev, 0.001), beta_2=0.0,
                            seed=seed)
    assert torch.equal(moments[3].cpu().view(torch.uint8).long(), exponent + 127)
    inside = torch.ones(n, dtype=torch.bool)
    inside[::BLOCK] = False  # (15 + h / 65536 of a step: 15 or, never, more)
    got = _values(moments[2], moments[3])
    bad = (got != want * 16 * scale) & inside
    assert not bad.any(), f'{int(bad.sum())} of {n} codes'
    assert torch.equal(got[::BLOCK], (15 * 16 * scale)[::BLOCK])
