"""Tensors that the AdamW function cannot update in place as what they stand for are refused, and nothing is written."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _call(dev, w, g=None, moments=None):
    from hgq2_amd import ops

    state = ops.adamw_state(dev, 0.1)
    try:
        ops.adamw_update_multi_([w], [torch.ones(8, device=dev) if g is None else g], [moments or ops.adamw_moments(8, dev)], state, decay=[0.5])
    finally:
        assert int(state[0]) in (0, 1)


def test_lazily_negated_variables_and_moments(dev):
    from hgq2_amd import ops

    base = -torch.ones(8, device=dev)
    with pytest.raises(ValueError, match='negated'):
        _call(dev, torch._neg_view(base))
    assert torch.equal(base, -torch.ones(8, device=dev))
    m, v = ops.adamw_moments(8, dev)
    with pytest.raises(ValueError, match='negated'):
        _call(dev, torch.ones(8, device=dev), moments=[torch._neg_view(m), v])
    assert not m.any() and not v.any()
    w = torch.ones(8, device=dev)
    _call(dev, w, g=torch._neg_view(-torch.ones(8, device=dev)))  # a gradient may be
    _call(dev, base.neg_(), g=torch.ones(8, device=dev))
    assert torch.equal(w, base)


@pytest.mark.parametrize('bits', [32, 8])
def test_moments_in_a_variables_memory(dev, bits):
    from hgq2_amd import ops

    buf = torch.ones(8, device=dev)
    m = ops.adamw_moments(8, dev, bits)
    m[0] = buf if bits == 32 else buf.view(torch.uint8)[:8].view(torch.float8_e4m3fn)
    with pytest.raises(ValueError, match='share memory'):
        _call(dev, buf, moments=m)
    assert torch.equal(buf, torch.ones(8, device=dev))
    with pytest.raises(ValueError, match='share memory'):
        ops.adamw_update_multi_([buf[:4], buf[4:]], [torch.ones(4, device=dev)] * 2, [ops.adamw_moments(4, dev), [buf[2:6], torch.zeros(4, device=dev)]],
                                ops.adamw_state(dev, 0.1))
    assert torch.equal(buf, torch.ones(8, device=dev))
