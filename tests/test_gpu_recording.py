"""Recording a training step while the graph of an eager step is alive: refused, and nothing has happened."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('optimizer', ['sgd', 'adamw'])
@pytest.mark.parametrize('how', ['step', 'warmup_data', 'feed', 'fit'])
def test_beside_a_living_loss(dev, optimizer, how):
    """The loss of an eager step keeps every variable's accumulating node, and with it that step's stream.  Variables, moments, the number of steps
    and the feed are as they were after the refusal, and once the loss is gone the same call works."""
    from hgq2_amd import ops
    from hgq2_amd.train import SGD, AdamW, GraphedTrainStep, ResidentBatches, fit, model_loss, train_step_for
    from hgq2_amd.utils.models import qdense_mlp

    torch.manual_seed(26)
    gen = torch.Generator().manual_seed(26)
    x, y = torch.randn(256, 16, generator=gen).to(dev), torch.randint(0, 5, (256,), generator=gen).to(dev)
    net = qdense_mlp(device=dev)
    net(x, training=False)
    make = {'sgd': lambda v: SGD(v, lr=0.01, fold_regularizers=True), 'adamw': lambda v: AdamW(v, fold_regularizers=True)}[optimizer]
    opt = make(net.parameters())
    opt.zero_grad()
    loss = model_loss(net, ops.sparse_ce(net(x, training=True), y), True)
    opt.backward(loss)
    opt.step()
    feed = ResidentBatches(x, y)
    feed.start_epoch(None)
    calls = {'step': lambda: GraphedTrainStep(net, ops.sparse_ce, opt, x[:64], y[:64]),
             'warmup_data': lambda: train_step_for(net, x[:64], y[:64], fused=False, optimizer=lambda v: opt, warmup_data=[(x[:64], y[:64])]),
             'feed': lambda: GraphedTrainStep(net, ops.sparse_ce, opt, x[:64], y[:64], feed=feed),
             'fit': lambda: fit(net, x, y, batch_size=64, fused=False, optimizer=lambda v: opt)}
    torch.cuda.synchronize()
    before = [p.detach().clone() for p in net.parameters()]
    moments = [m.clone() for m in opt._moments] if optimizer == 'adamw' else []
    with pytest.raises(RuntimeError, match='another stream that is still alive'):
        calls[how]()
    torch.cuda.synchronize()
    assert all(torch.equal(p, b) for p, b in zip(net.parameters(), before))
    if optimizer == 'adamw':
        assert opt.iterations == 1 and all(torch.equal(m, n) for m, n in zip(opt._moments, moments))
    at, labels = torch.empty_like(x[:64]), torch.empty_like(y[:64])
    feed.draw(at, labels)
    assert torch.equal(at, x[:64])  # the feed's first batch is still to come
    feed.start_epoch(None)
    del loss
    step = calls[how]()
    if how != 'fit':
        if how == 'step':
            step(x[:64], y[:64])
        else:
            step()
    torch.cuda.synchronize()
    assert all(torch.isfinite(p).all() for p in net.parameters()) and not all(torch.equal(p, b) for p, b in zip(net.parameters(), before))


def test_an_optimizer_of_the_callers_own(dev):
    """Anything with zero_grad, backward, step and fold_regularizers can be recorded, as before."""
    from hgq2_amd import ops
    from hgq2_amd.train import SGD, GraphedTrainStep
    from hgq2_amd.utils.models import qdense_mlp

    class Own:
        fold_regularizers = True

        def __init__(self, params):
            self.inner = SGD(params, lr=0.01, fold_regularizers=True)
            self.zero_grad, self.backward, self.step = self.inner.zero_grad, self.inner.backward, self.inner.step

    torch.manual_seed(27)
    gen = torch.Generator().manual_seed(27)
    x, y = torch.randn(64, 16, generator=gen).to(dev), torch.randint(0, 5, (64,), generator=gen).to(dev)
    net = qdense_mlp(device=dev)
    net(x, training=False)
    step = GraphedTrainStep(net, ops.sparse_ce, Own(net.parameters()), x, y)
    assert torch.isfinite(step()).all()
