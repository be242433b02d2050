"""Attention with relative positions, blocks on a residual stream and a teacher's top logits together, as a small student network is trained."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _scopes():
    from hgq2_amd.config import LayerConfigScope, QuantizerConfigScope

    return (QuantizerConfigScope(place='all', default_q_type='kbi', overflow_mode='SAT_SYM'), QuantizerConfigScope(place='datalane', default_q_type='kif', overflow_mode='WRAP'),
            LayerConfigScope(enable_ebops=True, beta0=1e-7))


def _student(positions=12, features=16, vocabulary=40, gated=True, buckets=8):
    from hgq2_amd.host import ResidualBlocks, Sequential
    from hgq2_amd.layers import QDense, QMultiHeadAttention

    a, b, c = _scopes()
    with a, b, c:
        blocks = [QMultiHeadAttention(num_heads=2, key_dim=8, relative_buckets=buckets, relative_max_distance=10, relative_initializer='glorot_uniform', name='attention'),
                  Sequential([QDense(24, activation='relu', name='up'), QDense(features, name='down')], name='wide')]
        gates = [QDense(features, name='gate'), None] if gated else None
        return Sequential([ResidualBlocks(blocks, gates, scale=0.5, name='blocks'), QDense(vocabulary, name='answers')], name='student')


def _data(dev, n=24, positions=12, features=16, vocabulary=40, top=5, seed=3):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, positions, features), generator=g)
    values, indices = (torch.randn((n, positions, vocabulary), generator=g) * 3).topk(top, dim=-1)
    indices[0, :, 2:] = -1
    return x.to(dev), (values.to(dev), indices.to(dev))


def test_attention_adds_the_bias_to_its_scores(dev):
    """The same projections, scores plus table[bucket] by indexing, the same softmax and combination: bit for bit; the table's gradient against
    autograd's through the indexing, where up to batch x positions terms meet in another order (96 u of their magnitudes on either side)."""
    from hgq2_amd import ops
    from hgq2_amd.layers import QMultiHeadAttention
    from hgq2_amd.layers.attn import mha

    a, b, c = _scopes()
    torch.manual_seed(5)
    with a, b, c:
        layer = QMultiHeadAttention(num_heads=3, key_dim=8, relative_buckets=12, relative_max_distance=9, relative_initializer='glorot_uniform')
        x = torch.randn(7, 21, 16, device=dev)
        layer(x)
        assert layer._relative_bias.shape == (12, 3)
        q, k, v = layer._query_dense(x), layer._key_dense(x), layer._value_dense(x)
        scores = ops.attn_scores(q, k).detach().requires_grad_(True)
        table = layer._relative_bias
        d = torch.arange(21)[None] - torch.arange(21)[:, None]
        first = torch.tensor(ops.relative_buckets(6, 9))
        bucket = ((d.abs()[..., None] >= first).sum(-1) + 6 * (d > 0)).to(dev)
        plain = table.detach().clone().requires_grad_(True)
        biased = (ops.relative_bias(scores, table, 9, True), scores + plain[bucket].permute(2, 0, 1))
        f = layer._softmax(biased[0])
        assert torch.equal(biased[0], biased[1]) and torch.equal(layer(x), layer._output_dense(ops.attn_combine(f, v)))
        got, want = (layer._softmax(t, training=True) for t in biased)
        assert torch.equal(got, want)
        dy = torch.randn(got.shape, device=dev)
        (ga,) = torch.autograd.grad(got, [table], dy, retain_graph=True)
        (gb,) = torch.autograd.grad(want, [plain], dy, retain_graph=True)
        (ds,) = torch.autograd.grad(got, [scores], dy)
        size = torch.zeros(12, 3, device=dev).index_add_(0, bucket.reshape(-1), ds.abs().sum(0).reshape(3, -1).t().contiguous())
        assert ga.abs().max() > 0 and ((ga - gb).abs() <= 2 * 96 * 2.0**-24 * size).all()
        # without a bias the layer is what it was
        with torch.no_grad():
            layer._relative_bias.zero_()
            zero = layer(x)
        plain_layer = QMultiHeadAttention(num_heads=3, key_dim=8)
        plain_layer(x)
        for p, s in zip(plain_layer.parameters(), [t for t in layer.parameters() if t is not layer._relative_bias]):
            p.data.copy_(s)
        keep, mha.FUSED = mha.FUSED, False
        try:
            with torch.no_grad():
                assert torch.equal(plain_layer(x), zero)
        finally:
            mha.FUSED = keep


@pytest.mark.parametrize('positions', [64, 65, 90])
def test_attention_of_more_positions_and_masks(dev, positions):
    """Up to 64 positions the scores come from the contraction kernels, beyond from the library: the bias is added to either, and a masked key
    gets no weight whatever its bias."""
    from hgq2_amd.layers import QMultiHeadAttention

    a, b, c = _scopes()
    torch.manual_seed(6)
    with a, b, c:
        layer = QMultiHeadAttention(num_heads=2, key_dim=8, relative_buckets=8, relative_max_distance=30, relative_bidirectional=False)
        x = torch.randn(3, positions, 16, device=dev)
        layer(x)
        with torch.no_grad():
            layer._relative_bias.copy_(torch.randn(8, 2, device=dev))
            out, scores = layer(x, use_causal_mask=True, return_attention_scores=True)
        assert torch.isfinite(out).all() and not scores.triu(1).any() and scores[..., 0, 0].any()


def test_blocks_on_a_residual_stream(dev):
    """The layer against its formula in 64 bits on the blocks' own outputs, float32 roundings apart (a norm of 16 channels: 40 u of each value is far
    more than its sums and products lose, times what two norms pass on)."""
    torch.manual_seed(7)
    model = _student()
    x, _ = _data(dev)
    model(x)
    layer = model.layers[0]
    norm = lambda t, g: t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * g.double()  # noqa: E731
    with torch.no_grad():
        for p in layer._parameters.values():
            p.copy_(1 + 0.2 * torch.randn_like(p))
        s = x.double()
        h = norm(s, layer._var_gamma_0)
        g = layer.gates[0](h.float()).double().sigmoid()
        u = layer.blocks[0](h.float()).double()
        s = s + 0.5 * g * norm(u, layer._var_post_0)
        from hgq2_amd import ops

        y, h1 = ops.residual_norm(x, u.float(), layer._var_post_0, layer._var_gamma_1, layer.gates[0](h.float()), 'sigmoid', 0.5)
        assert ((y - s).abs() <= 40 * 2.0**-24 * (s.abs() + 1)).all() and ((h1 - norm(s, layer._var_gamma_1)).abs() <= 200 * 2.0**-24 * (h1.abs() + 1)).all()
        u2 = layer.blocks[1](h1)
        want = norm(y.double() + 0.5 * norm(u2.double(), layer._var_post_1), layer._var_gamma_2)
        # (the layer's own first norm may round h otherwise than this one, and a quantizer makes a step of its own of that)
        _, got = ops.residual_norm(y, u2, layer._var_post_1, layer._var_gamma_2, None, None, 0.5)
        assert ((got - want).abs() <= 200 * 2.0**-24 * (want.abs() + 1)).all()
        out = layer(x)
        assert out.shape == x.shape and torch.isfinite(out).all()
        a = ops.rms_norm(x, layer._var_gamma_0)
        b, c = ops.residual_norm(x, layer.blocks[0](a), layer._var_post_0, layer._var_gamma_1, layer.gates[0](a), 'sigmoid', 0.5)
        _, d = ops.residual_norm(b, layer.blocks[1](c), layer._var_post_1, layer._var_gamma_2, None, None, 0.5)
        assert torch.equal(out, d)


@pytest.mark.parametrize('how', ['distill_topk', 'callable'])
def test_trained_in_a_recorded_step(dev, how):
    """Five steps recorded and replayed against the same five steps launched one by one: the same bits in losses and variables; every variable of the
    blocks, and the bias table, is trained."""
    from hgq2_amd import ops
    from hgq2_amd.train import SGD, model_loss, train_step_for

    x, y = _data(dev)
    loss = 'distill_topk' if how == 'distill_topk' else lambda out, t: 2.0 * ops.distill_topk(out, *t, temperature=2.0)
    models = []
    for _ in range(2):
        torch.manual_seed(9)
        models.append(_student())
        models[-1](x)
    model, twin = models
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    step = train_step_for(model, x, y, lr=0.02, loss=loss, warmup=2)
    assert step.path == 'layers_graph'
    got = [float(step(x, y)) for _ in range(3)]
    opt = SGD(twin.parameters(), lr=0.02, fold_regularizers=True)
    want = []
    for _ in range(5):
        with ops.overlap_ebops():
            opt.zero_grad(set_to_none=True)
            out = twin(x, training=True)
            total = model_loss(twin, ops.distill_topk(out, *y) if how == 'distill_topk' else loss(out, y), True)
            opt.backward(total)
            opt.step()
        want.append(float(total.detach()))
    assert got == want[2:] and all(math.isfinite(v) for v in got)
    for (n, p), q in zip(model.named_parameters(), twin.parameters()):
        assert torch.equal(p, q), n
    for n in ('layers.0._var_gamma_0', 'layers.0._var_gamma_1', 'layers.0._var_gamma_2', 'layers.0._var_post_0', 'layers.0._var_post_1', 'layers.0.blocks.0._var_relative_bias'):
        assert not torch.equal(dict(model.named_parameters())[n], before[n]), n


def test_fit_with_a_teachers_lists(dev):
    """Targets of several tensors, shuffled, with a last batch that is shorter: each batch is trained on once, as the same loop written out does."""
    from hgq2_amd import ops
    from hgq2_amd.train import fit

    x, (values, indices) = _data(dev, n=53)
    lse = torch.logsumexp(values, -1) + 0.2
    weight = torch.ones_like(lse)
    weight[:, -3:] = 0
    torch.manual_seed(10)
    model = _student()
    model(x[:20])
    seen = []

    def loss(out, y):
        seen.append(tuple(y[0].shape))
        return ops.distill_topk(out, y[0], y[1], teacher_lse=y[2], sample_weight=y[3])

    logs = fit(model, x, (values, indices, lse, weight), loss=loss, batch_size=20, epochs=2, lr=0.01, seed=4)
    assert len(logs) == 2 and all(math.isfinite(e['loss']) for e in logs)
    assert {s[0] for s in seen} == {20, 13}
    logs = fit(model, x, (values, indices, lse, None), loss='distill_topk', batch_size=53, epochs=1, lr=0.01)
    assert math.isfinite(logs[0]['loss'])
    with pytest.raises(ValueError, match='same, non-zero number'):
        fit(model, x, (values[:5], indices), loss='distill_topk')


def test_saved_and_loaded(dev, tmp_path):
    from hgq2_amd.host import RMSNormalization, Sequential
    from hgq2_amd.saving import load_model, save_model, variable_paths

    torch.manual_seed(11)
    model = Sequential([RMSNormalization(epsilon=1e-5, name='norm'), _student()], name='saved')
    x, _ = _data(dev)
    model(x)
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() and p.requires_grad:
                p.add_(0.05 * torch.rand_like(p))
    paths = variable_paths(model)
    assert 'saved/student/blocks/attention/relative_bias' in paths and 'saved/norm/scale' in paths and 'saved/student/blocks/gamma_2' in paths
    save_model(model, tmp_path / 'model.npz')
    again = load_model(tmp_path / 'model.npz')
    with torch.no_grad():
        assert torch.equal(model(x), again(x))


def test_from_two_threads(dev):
    """Calls of two threads at once, on streams of their own: each gets what it gets alone."""
    import threading

    from hgq2_amd import ops

    g = torch.Generator().manual_seed(12)
    x, u = torch.randn((300, 700), generator=g).to(dev), torch.randn((300, 700), generator=g).to(dev)
    s, t = torch.randn((4, 2, 40, 40), generator=g).to(dev), torch.randn((8, 2), generator=g).to(dev)
    i = torch.randint(0, 700, (300, 9), generator=g).to(dev)

    def run():
        a, b, c, d = (v.clone().requires_grad_(True) for v in (x, u, s, t))
        y, h = ops.residual_norm(a, b)
        loss = ops.distill_topk(h, u[:, :9].detach(), i)
        out = ops.relative_bias(c, d, 30)
        return [v.detach() for v in (y, h, loss, out, *torch.autograd.grad(loss, [a, b]), *torch.autograd.grad(out.square().sum(), [c, d]))]

    want, got = run(), {}
    torch.cuda.synchronize()

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got[k] = run()
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for k in range(2):
        assert all(torch.equal(a, b) for a, b in zip(want, got[k]))
