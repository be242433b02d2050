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


def test_the_clipping_factor_is_keras(dev):
    """clipnorm times the rounded reciprocal of the rounded norm.  With beta_1 = 0 the first moment is the clipped gradient, and of a gradient of
    one that is the factor itself."""
    from hgq2_amd import ops

    gen = torch.Generator().manual_seed(32)
    other = 30 * torch.rand(200, generator=gen)
    clips = (0.9 * torch.rand(200, generator=gen) + 0.05).tolist()
    clips[:4] = [0.1, 0.3, 0.7, 1.0]
    got, want = [], []
    for a, clip in zip(other.tolist(), clips):
        g = torch.tensor([1.0, a])
        m, norm = ops.adamw_moments(2, dev), torch.zeros((), device=dev)
        ops.adamw_update_multi_([torch.zeros(2, device=dev)], [g.to(dev)], [m], ops.adamw_state(dev, 0.001), beta_1=0.0, clipnorm=clip, norm_out=norm)
        n = np.float32(np.sqrt(np.sum(g.double().numpy() ** 2)))
        assert np.float32(norm.item()) == n
        got.append(m[0][0].item())
        want.append(float(np.float32(clip) * (np.float32(1) / n)) if n > np.float32(clip) else 1.0)
    assert got == want


@pytest.mark.parametrize('norm,clip', [(2.0**-130, 2.0**-133), (2.0**-130, 2.0**-126), (2.0**127, 2.0**100), (1.5 * 2.0**127, 3 * 2.0**80), (2.0**-126, 2.0**-128)])
def test_clipping_at_the_ends_of_the_range(dev, norm, clip):
    """Where the reciprocal overflows or is no normal number the factor is the quotient, here a power of two."""
    from hgq2_amd import ops

    m = ops.adamw_moments(1, dev)
    ops.adamw_update_multi_([torch.zeros(1, device=dev)], [torch.tensor([norm], device=dev)], [m], ops.adamw_state(dev, 0.001), beta_1=0.0, clipnorm=clip)
    assert m[0].item() == min(norm, clip)
