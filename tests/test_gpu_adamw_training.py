"""A quantized network trained with AdamW by three ways: recorded, eager with gradient pieces beside the variables, and through autograd's
accumulation.  The first two launch the same, so their bits are compared; the third adds a variable's pieces in another order."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
LR, DECAY, EPS = 0.002, 0.004, 1e-7


def _networks(dev, count):
    from hgq2_amd.utils.models import qdense_mlp

    gen = torch.Generator().manual_seed(31)
    x, y = torch.randn(512, 16, generator=gen).to(dev), torch.randint(0, 5, (512,), generator=gen).to(dev)
    torch.manual_seed(31)
    nets = [qdense_mlp(device=dev) for _ in range(count)]
    for net in nets:
        net(x, training=False)
    for net in nets[1:]:
        with torch.no_grad():
            for a, b in zip(net.parameters(), nets[0].parameters()):
                a.copy_(b)
    return nets, x, y


@pytest.mark.parametrize('clip', [None, 1.0])
@pytest.mark.parametrize('bits', [32, 8])
def test_recorded_and_eager_steps_have_the_same_bits(dev, bits, clip):
    from hgq2_amd import ops
    from hgq2_amd.train import AdamW, model_loss, train_step_for

    make = lambda v: AdamW(v, lr=LR, global_clipnorm=clip, state_bits=bits, seed=4, fold_regularizers=True)  # noqa: E731
    (a, b), x, y = _networks(dev, 2)
    step = train_step_for(a, x, y, optimizer=make, warmup=1)
    losses = [float(step()) for _ in range(4)]
    opt = make(b.parameters())
    pieces = 0
    for k in range(5):
        opt.zero_grad()
        loss = model_loss(b, ops.sparse_ce(b(x, training=True), y), True)
        opt.backward(loss)
        pieces += sum(len(getattr(p, '_hgq_side', None) or ()) for p in opt.params)
        opt.step()
        if k:
            assert float(loss.detach()) == losses[k - 1], k
    assert pieces > 0
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q) and torch.isfinite(p).all()
    for m, n in zip(step.opt._moments, opt._moments):
        assert torch.equal(m.view(torch.uint8), n.view(torch.uint8))
    assert step.opt.iterations == opt.iterations == 5


def test_pieces_and_accumulated_gradients_agree(dev):
    """One step.  A gradient of k terms is off by (k - 1) u times the sum of their magnitudes in either order, so two of them by twice that; the
    products with a scale add u each.  m is the gradient times 1 - beta_1 (off by 3 u besides), and the first step is lr g / (|g| + eps / sqrt(1 -
    beta_2)), whose slope is at most lr / (|g| + that); 16 u of the step for the roundings in between, 3 u of w."""
    from hgq2_amd import ops
    from hgq2_amd.train import AdamW, model_loss

    (a, b), x, y = _networks(dev, 2)
    start = [p.detach().clone() for p in a.parameters()]
    opts = [AdamW(net.parameters(), lr=LR, weight_decay=DECAY, epsilon=EPS) for net in (a, b)]
    for k, (net, opt) in enumerate(zip((a, b), opts)):
        opt.zero_grad()
        loss = model_loss(net, ops.sparse_ce(net(x, training=True), y))
        (opt.backward(loss) if k == 0 else loss.backward())
    terms, many = [], 0
    for p in opts[0].params:
        side = [d.double().reshape(p.shape) * (1.0 if s is None else s.double()) for s, d in getattr(p, '_hgq_side', None) or ()]
        terms.append(([] if p.grad is None else [p.grad.double()]) + side)
        many += len(side) > 0
    assert many >= 6  # bit-width variables of every layer
    for opt in opts:
        opt.step()
    by_id = {id(p): w for p, w in zip(a.parameters(), start)}
    for k, (p, q, t) in enumerate(zip(opts[0].params, opts[1].params, terms)):
        assert q.grad is not None and not getattr(q, '_hgq_side', None)
        total, size = sum(t), sum(v.abs() for v in t)
        off = 2 * (len(t) + 1) * U * size
        name = f'{getattr(p, "var_name", "")} ({len(t)} terms)'
        assert ((q.grad.double() - total).abs() <= off).all(), name
        part = slice(opts[0].offsets[k], opts[0].offsets[k] + p.numel())
        m = [opt.momentum[part].double().view(p.shape) for opt in opts]
        for have in m:
            assert ((have - 0.1 * total).abs() <= 0.1 * (off + 4 * U * size)).all(), name
        w0, rest = by_id[id(p)].double(), EPS / math.sqrt(0.001)
        stepped = LR * total / (total.abs() + rest)
        want = w0 * (1 - LR * DECAY) - stepped
        c = getattr(p, 'constraint', None)
        if c is not None and c.bounds() is not None:
            want = want.clamp(*c.bounds())
        tol = LR * (off + 4 * U * size) / (total.abs() + rest) + 16 * U * stepped.abs() + 3 * U * w0.abs()
        for have in (p, q):
            assert ((have.detach().double() - want).abs() <= tol).all(), name
