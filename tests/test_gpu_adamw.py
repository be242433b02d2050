"""The AdamW step and the global gradient norm against a plain implementation in 64 bits.

Tolerances follow the arithmetic of one step from exact inputs, u = 2^-24 (half a step of fp32).  The clipping factor is off by at
most 2 u (the norm's rounding and the division's), so the gradient by 3 u.  m: the gradient and three roundings of the difference, times
1 - beta_1, and one of the sum: 6 u (1 - beta_1) (|g| + |m|) + u |m'|.  v: g g is off by 7 u, then the same: 10 u (1 - beta_2) (g^2 + v) +
u v'.  The step m alpha / (r + eps): what m and half of what v are off
by, relatively, and seven roundings: root, sum, alpha and two products u each, the reciprocal a unit in the last place, 2 u.  w: that, and three roundings of w; a 16-bit
type adds half a step of its own."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
BLOCK = 256
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def _philox(blocks, step, seed):
    mask = np.uint64(0xFFFFFFFF)
    c = [blocks & mask, blocks >> np.uint64(32), np.full_like(blocks, step & 0xFFFFFFFF), np.full_like(blocks, step >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(7):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & mask, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & mask]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, axis=1).reshape(-1)


def _values(codes, scales):
    """The numbers that codes and scales stand for, in 64 bits."""
    c = codes.cpu().view(torch.uint8).long()
    e, f = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, f * 2.0**-9, (8 + f) * torch.pow(2.0, (e - 10).double()))
    v = torch.where((c & 127) == 127, torch.nan, v) * torch.where(c >= 128, -1.0, 1.0)
    s = torch.pow(2.0, scales.cpu().view(torch.uint8).double() - 127)
    return v * s.repeat_interleave(BLOCK)[:v.numel()]


def _plain(w, g, m, v, t, lr=0.001, b1=0.9, b2=0.999, eps=1e-7, decay=0.004, c=1.0, l1=0.0, lo=-math.inf, hi=math.inf):
    """One step in 64 bits on the CPU: (w, m, v, tolerances of the three)."""
    w, g, m, v = (k.detach().double().cpu().reshape(-1) for k in (w, g, m, v))
    g = (g + l1) * c
    alpha = lr * math.sqrt(1 - b2**t) / (1 - b1**t)
    tm, tv = 6 * U * (1 - b1) * (g.abs() + m.abs()), 10 * U * (1 - b2) * (g * g + v)
    m, v = m + (g - m) * (1 - b1), v + (g * g - v) * (1 - b2)
    tm, tv = tm + U * m.abs(), tv + U * v
    r = v.sqrt()
    step = m * alpha / (r + eps)
    new = w * (1 - lr * decay) - step
    tw = 3 * U * w.abs() + alpha * tm / (r + eps) + step.abs() * (tv / (2 * v).clamp(min=1e-300) + 7 * U)
    tw = torch.where(v == 0, 3 * U * w.abs(), tw)
    return new.clamp(lo, hi), m, v, tw, tm, tv


def _near(got, want, tol, dtype, what):
    got, want = got.detach().double().cpu().reshape(-1), want.reshape(-1)
    tol = tol + HALF[dtype] * (want.abs() + tol) + (2.0**-25 if dtype == torch.float16 else 0.0)  # (half the spacing below fp16's normals)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()}, worst {float(((got - want).abs() / tol.clamp(min=1e-300)).max()):.3g} times the tolerance'


def _codes_near(codes, scales, want, tol, h, floor, what):
    """Codes and scales against the stochastic rounding of ``want`` (64 bits) with the 16-bit numbers ``h``."""
    n = want.numel()
    pad = -n % BLOCK
    rows = torch.cat([want, want.new_zeros(pad)]).view(-1, BLOCK).abs()
    trows = torch.cat([tol, tol.new_zeros(pad)]).view(-1, BLOCK)
    most = rows.max(dim=1).values
    s = torch.where(most > 0, torch.frexp(most)[1].double() - 1 + 127 - 7, 1.0).clamp(min=1)
    have = scales.cpu().view(torch.uint8).double()
    # another scale only where the block's largest is within its tolerance of a power of two
    at = rows.argmax(dim=1, keepdim=True)
    slack = trows.gather(1, at).squeeze(1)
    edge = torch.minimum(most - torch.pow(2.0, s + 7 - 127), torch.pow(2.0, s + 8 - 127) - most).abs() <= slack
    assert ((have == s) | edge).all(), f'{what}: scales'
    keep = (have == s).repeat_interleave(BLOCK)[:n]
    scale = torch.pow(2.0, s - 127).repeat_interleave(BLOCK)[:n]
    q = want.abs() / scale
    unit = torch.pow(2.0, torch.frexp(q)[1].double().clamp(min=-5) - 4)
    x = q / unit + torch.from_numpy(h.astype(np.float64)) / 65536
    y = torch.floor(x) * unit
    y = torch.where((want != 0) & (y == 0) & floor, 2.0**-9, y)
    got = _values(codes, torch.full((-(-n // BLOCK),), 127, dtype=torch.uint8)).abs()
    # the neighbouring code only where the sum is within the tolerance (and the 2^-20 of the subnormal codes) of a whole number
    close = (x - torch.round(x)).abs() <= tol / scale / unit + 2.0**-20
    ok = (got == y) | (close & ((got - y).abs() <= unit * 1.001)) | ~keep
    assert ok.all(), f'{what}: {int((~ok).sum())} of {n} codes'
    assert (close & keep).double().mean() < 0.01  # (the exemption stays an exemption)
    sign = codes.cpu().view(torch.uint8) >= 128
    assert ((sign == (want < 0)) | (want.abs() <= tol)).all(), f'{what}: signs'


def _variables(sizes, dtype, dev, seed, odd=False):
    """Variables and gradients; ``odd``: views that begin one element behind an aligned address, with guards around them."""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        w, g = torch.randn(n, generator=gen) * 0.1, torch.randn(n, generator=gen) * 10.0 ** float(torch.randint(-3, 2, (1,), generator=gen))
        pair = []
        for k in (w, g):
            buf = torch.full((n + 16,), 7.0, dtype=dtype, device=dev)
            at = 9 if odd else 8
            buf[at:at + n] = k.to(dtype).to(dev)
            pair.append((buf, buf[at:at + n]))
        out.append(pair)
    return out


SIZES = {'few': [1, 3, 255, 256, 257], 'many': [5 + 37 * k for k in range(61)], 'none': [4, 0, 9], 'long': [(1 << 22) + (1 << 20) + 3],
         'vast': [17_000_003, 4099, 5]}  # (more than the card's cache holds)


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('sizes,odd,clip', [('few', False, None), ('few', True, 0.5), ('many', False, 0.5), ('none', False, 1e6), ('long', False, 0.5),
                                            ('long', True, None)])
def test_two_steps_against_64_bits(dev, sizes, odd, clip, dtype, bits):
    _two_steps(dev, sizes, odd, clip, dtype, bits)


@pytest.mark.parametrize('dtype,bits,clip', [(torch.float32, 32, 0.5), (torch.float32, 8, 0.5), (torch.float32, 8, None), (torch.bfloat16, 32, None)])
def test_more_than_the_cache_holds(dev, dtype, bits, clip):
    _two_steps(dev, 'vast', False, clip, dtype, bits)


def _two_steps(dev, sizes, odd, clip, dtype, bits):
    from hgq2_amd.train import AdamW

    pairs = _variables(SIZES[sizes], dtype, dev, len(sizes) + bits, odd)
    params = [torch.nn.Parameter(w) for (_, w), _ in pairs]
    for p, (_, (_, g)) in zip(params, pairs):
        p.grad = g
    opt = AdamW(params, lr=0.01, global_clipnorm=clip, state_bits=bits, seed=12345678901)
    total = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params))
    c = 1.0 if clip is None else min(1.0, clip / total)
    for t in (1, 2):
        old = [p.detach().clone() for p in params]
        if bits == 32:
            before = [opt.momentum.clone(), opt.velocity.clone()]
        else:
            before = [_values(opt.momentum, opt.momentum_scale), _values(opt.velocity_root, opt.velocity_scale) ** 2]
        opt.step()
        if clip is not None:
            assert abs(float(opt.grad_norm) - total) <= 2 * U * total
        for k, (p, w0) in enumerate(zip(params, old)):
            n, at = p.numel(), opt.offsets[k]
            if not n:
                continue
            part = slice(at, at + n)
            w, m, v, tw, tm, tv = _plain(w0, p.grad, before[0][part], before[1][part], t, lr=0.01, c=c)
            _near(p, w, tw, dtype, f'w of {n}')
            if bits == 32:
                _near(opt.momentum[part], m, tm, torch.float32, f'm of {n}')
                _near(opt.velocity[part], v, tv, torch.float32, f'v of {n}')
            else:
                h = _philox(np.arange(at // 4, (at + n + 3) // 4, dtype=np.uint64), t, 12345678901)[:n]
                r = v.sqrt()
                blocks = slice(at // BLOCK, at // BLOCK + -(-n // BLOCK))
                _codes_near(opt.momentum[part], opt.momentum_scale[blocks], m, tm, h & np.uint64(0xFFFF), False, f'm of {n}, step {t}')
                _codes_near(opt.velocity_root[part], opt.velocity_scale[blocks], r, tv / (2 * r).clamp(min=1e-300) + 2 * U * r, h >> np.uint64(16), True,
                            f'r of {n}, step {t}')
    assert opt.iterations == 2
    for (wb, w), (gb, g) in pairs:  # nothing written beside the variables, nothing in the gradients
        at = w.storage_offset()
        for b in (wb, gb):
            assert (b[:at] == 7).all() and (b[at + w.numel():] == 7).all()


@pytest.mark.parametrize('bits', [32, 8])
def test_a_recorded_step_counts_on(dev, bits):
    """Replays are further steps, with the learning rate and gradients of their time; another graph shares nothing but the optimizer."""
    from hgq2_amd.train import AdamW

    gen = torch.Generator().manual_seed(3)
    start = [torch.randn(n, generator=gen).to(dev) for n in (700, 33, 4096)]
    grads = [torch.zeros_like(k) for k in start]
    feeds = [[torch.randn(k.shape, generator=gen).to(dev) for k in start] for _ in range(8)]
    rates = [1e-3, 1e-3, 1e-2, 1e-2, 3e-4, 3e-4, 1e-3, 1e-3]

    def make():
        params = [torch.nn.Parameter(k.clone()) for k in start]
        for p, g in zip(params, grads):
            p.grad = g
        return params, AdamW(params, lr=rates[0], global_clipnorm=0.7, state_bits=bits, seed=5)

    params, opt = make()
    twin_params, twin = make()
    graphs = []
    for g, f in zip(grads, feeds[0]):
        g.copy_(f)
    opt.step(), twin.step()
    side = torch.cuda.Stream()
    for _ in range(2):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            opt.step()
        graphs.append(graph)
    for k in range(1, 8):
        for g, f in zip(grads, feeds[k]):
            g.copy_(f)
        opt.lr = twin.lr = rates[k]
        graphs[k % 2].replay()
        twin.step()
        torch.cuda.synchronize()
        assert opt.iterations == twin.iterations == k + 1
        for a, b in zip(params, twin_params):
            assert torch.equal(a, b), k
        assert torch.equal(opt.grad_norm, twin.grad_norm)
        for name in opt._names:
            assert torch.equal(getattr(opt, name).view(torch.uint8), getattr(twin, name).view(torch.uint8)), (k, name)
    with pytest.raises(RuntimeError, match='capture'):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            opt.lr = 1.0


@pytest.mark.parametrize('bits', [32, 8])
def test_continuing_from_a_state(dev, bits):
    from hgq2_amd.train import AdamW

    gen = torch.Generator().manual_seed(4)
    start, grad = torch.randn(1000, generator=gen).to(dev), torch.randn(1000, generator=gen).to(dev)

    def make(w):
        p = torch.nn.Parameter(w.clone())
        p.grad = grad
        return p, AdamW([p], state_bits=bits, seed=9)

    p, opt = make(start)
    for _ in range(3):
        opt.step()
    q, other = make(p.detach())
    other.load_state_dict(opt.state_dict())
    for _ in range(2):
        opt.step(), other.step()
    assert torch.equal(p, q) and opt.iterations == other.iterations == 5
    state = opt.state_dict()
    with pytest.raises(ValueError, match='expected'):
        other.load_state_dict({**state, 'momentum': state['momentum'][:-1]})
    with pytest.raises(ValueError, match='entries'):
        other.load_state_dict({k: v for k, v in state.items() if k != 'momentum'})
    with pytest.raises(ValueError, match='negative'):
        other.load_state_dict({**state, 'iterations': -1})


def test_pieces_regularizers_and_constraints(dev):
    """Gradient pieces with and without a scale, a folded regularizer, bounds, a variable without decay, one without a gradient, strided gradients."""
    from hgq2_amd.constraints import MinMax
    from hgq2_amd.regularizers import MonoL1
    from hgq2_amd.train import AdamW

    gen = torch.Generator().manual_seed(6)
    rnd = lambda *s: torch.randn(*s, generator=gen).to(dev)  # noqa: E731
    params = [torch.nn.Parameter(rnd(20, 30)) for _ in range(5)]
    a, b, c, d, e = params
    scale = torch.tensor([0.375], device=dev)
    a.grad, a._hgq_side = rnd(20, 30), [(scale, rnd(600)), (None, rnd(600))]
    b._hgq_side = [(None, rnd(600)) for _ in range(6)]  # (more than a descriptor holds)
    b.regularizer, b.constraint = MonoL1(0.25), MinMax(-0.5, 0.5)
    c.grad = rnd(30, 20).t()
    d.grad, d.var_name = rnd(20, 30), 'bn_gamma'
    opt = AdamW(params, lr=0.01, weight_decay=0.1, fold_regularizers=True, global_clipnorm=3.0)
    opt.exclude_from_weight_decay(var_names=['gamma'])
    old = [p.detach().clone() for p in params]
    total = [a.grad + (scale * a._hgq_side[0][1] + a._hgq_side[1][1]).view(20, 30), sum(s for _, s in b._hgq_side).view(20, 30) + 0.25, c.grad, d.grad]
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in total))
    opt.step()
    # (up to six pieces add five roundings of sums no larger than the sum of their magnitudes, here at most 8 times the gradient's scale of 1)
    assert abs(float(opt.grad_norm) - norm) <= 64 * U * norm
    for k, (p, g, decay, lim) in enumerate(zip(params, total, (0.1, 0.1, 0.1, 0.0), (math.inf, 0.5, math.inf, math.inf))):
        w, _, _, tw, _, _ = _plain(old[k], g.reshape(-1), torch.zeros(600), torch.zeros(600), 1, lr=0.01, decay=decay, c=3.0 / norm, lo=-lim, hi=lim)
        # the first step is lr sign(g): the pieces' rounding shows where g is near zero, against epsilon
        gc = (g.double().cpu().reshape(-1) * 3.0 / norm).abs()
        tw = tw + 0.01 * 64 * U * 8 / (gc + 1e-7 / math.sqrt(0.001))
        _near(p, w, tw, torch.float32, f'variable {k}')
    assert torch.equal(e, old[4])
    assert float(b.detach().abs().max()) == 0.5
    opt.zero_grad()
    assert a.grad is None and b._hgq_side is None
    opt.step()  # no gradients at all: nothing happens
    assert opt.iterations == 1


def test_what_is_not_finite(dev):
    """A NaN or an infinity stays with its element without clipping; with it, every variable becomes NaN; 8-bit codes hold the NaN alone."""
    from hgq2_amd.train import AdamW

    for bad in (float('nan'), float('inf'), -float('inf')):
        for bits in (32, 8):
            g = torch.ones(600, device=dev)
            g[37] = bad
            p = torch.nn.Parameter(torch.ones(600, device=dev))
            p.grad = g
            opt = AdamW([p], state_bits=bits)
            opt.step()
            finite = torch.isfinite(p)
            assert not finite[37] and int(finite.sum()) == 599
            if bits == 8:
                codes = opt.momentum.view(torch.uint8)[:600].cpu()
                assert (codes[37] & 127) == 127 and int(((codes & 127) == 127).sum()) == 1
            opt.step()
            assert int(torch.isfinite(p).sum()) == 599
            q = torch.nn.Parameter(torch.ones(600, device=dev))
            q.grad = g
            AdamW([q], state_bits=bits, global_clipnorm=1.0).step()
            assert torch.isnan(q).all()
    # gradients whose squares leave fp32 have a finite norm
    p = torch.nn.Parameter(torch.zeros(8, device=dev))
    p.grad = torch.full((8,), 1e30, device=dev)
    opt = AdamW([p], global_clipnorm=1.0)
    opt.step()
    assert abs(float(opt.grad_norm) / (1e30 * math.sqrt(8)) - 1) < 1e-6 and torch.isfinite(p).all()
    p.grad = torch.zeros(8, device=dev)
    opt.step()
    assert float(opt.grad_norm) == 0 and torch.isfinite(p).all()


def test_slow_averages_move_in_8_bits(dev):
    """A constant gradient g: r approaches |g| as sqrt(1 - beta_2^t), although one step is far below half a code.  Rounding leaves r within
    about a fifth of it (code distances of 1/16 to 1/8 against steps of 1/2000); the mean over 8192 elements then lies within a
    hundredth, and five are allowed."""
    from hgq2_amd.train import AdamW

    gen = torch.Generator().manual_seed(8)
    g = (torch.rand(8192, generator=gen) + 0.5).to(dev)
    p = torch.nn.Parameter(torch.zeros(8192, device=dev))
    p.grad = g
    opt = AdamW([p], state_bits=8, seed=1)
    for t in range(1, 2001):
        opt.step()
        if t in (30, 300, 2000):
            r = _values(opt.velocity_root, opt.velocity_scale) / g.double().cpu()
            m = _values(opt.momentum, opt.momentum_scale) / g.double().cpu()
            assert abs(float(r.square().mean()) / (1 - 0.999**t) - 1) < 0.1, t  # (of the squares: twice as much)
            assert abs(float(m.mean()) / (1 - 0.9**t) - 1) < 0.05, t


def test_global_norm(dev):
    from hgq2_amd import ops

    gen = torch.Generator().manual_seed(9)
    for sizes in ([1], [0], [0, 5], [3, 1000, 2047, 2048, 2049], [17] * 100, [3_000_001]):
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            ts = [torch.randn(n, generator=gen).to(dtype).to(dev) for n in sizes]
            want = math.sqrt(sum(float(t.double().square().sum()) for t in ts))
            got = ops.global_norm(ts)
            assert got.dtype == torch.float32 and got.dim() == 0
            assert abs(float(got) - want) <= (U + 1e-12) * want  # one rounding to fp32, and those of fp64
    mixed = [torch.ones(4, 6, device=dev).t(), None, torch.full((5,), 2.0, dtype=torch.float16, device=dev)]
    assert float(ops.global_norm(mixed)) == math.sqrt(44) or abs(float(ops.global_norm(mixed)) - math.sqrt(44)) <= U * 8
    big = torch.randn(1_000_003, generator=gen).to(dev)
    assert len({float(ops.global_norm([big, big[1:]])) for _ in range(5)}) == 1
    with pytest.raises(ValueError, match='float32'):
        ops.global_norm([torch.zeros(3, dtype=torch.float64, device=dev)])


def test_update_on_given_tensors(dev):
    """The function under the class: own moments and state, another stream, refusals."""
    from hgq2_amd import ops

    gen = torch.Generator().manual_seed(10)
    w, g = torch.randn(500, generator=gen).to(dev), torch.randn(500, generator=gen).to(dev)
    w0 = w.clone()
    moments, state, norm = ops.adamw_moments(500, dev), ops.adamw_state(dev, 0.01), torch.zeros((), device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.adamw_update_multi_([w], [g], [moments], state, decay=[0.1], l1=[0.5], lo=[-1.0], hi=[1.0], clipnorm=2.0, norm_out=norm)
    s.synchronize()
    want = float((g.double() + 0.5).square().sum().sqrt())
    assert abs(float(norm) - want) <= 4 * U * want
    new, m, _, tw, tm, _ = _plain(w0, g, torch.zeros(500), torch.zeros(500), 1, lr=0.01, decay=0.1, c=2.0 / want, l1=0.5, lo=-1.0, hi=1.0)
    tw = tw + 0.01 * 8 * U * 2 / ((g.double().cpu() + 0.5).abs() * 2.0 / want + 1e-7 / math.sqrt(0.001))  # (the rounding of g + l1 near zero)
    _near(w, new, tw, torch.float32, 'w')
    _near(moments[0], m, tm + 2 * U, torch.float32, 'm')
    for args in (([w, w], [g, g], [moments, moments]), ([w], [g[:-1]], [moments]), ([w], [g.double()], [moments]),
                 ([w], [g], [ops.adamw_moments(499, dev)]), ([w], [g.cpu()], [moments]), ([w.view(20, 25).t()], [g.view(25, 20)], [moments])):
        with pytest.raises(ValueError):
            ops.adamw_update_multi_(*args, state)
    with pytest.raises(ValueError, match='state'):
        ops.adamw_update_multi_([w], [g], [moments], state[:4])


def _model(dev):
    from hgq2_amd.utils.models import qdense_mlp

    torch.manual_seed(11)
    return qdense_mlp(device=dev)


@pytest.mark.parametrize('bits', [32, 8])
def test_in_a_training_step(dev, bits):
    """A quantized network trained with AdamW: the recorded step, the eager step with gradient pieces left beside the variables, and the
    eager step through autograd's accumulation go the same way."""
    from hgq2_amd import ops
    from hgq2_amd.train import AdamW, model_loss, train_step_for

    gen = torch.Generator().manual_seed(12)
    x, y = torch.randn(512, 16, generator=gen).to(dev), torch.randint(0, 5, (512,), generator=gen).to(dev)
    make = lambda v: AdamW(v, lr=0.002, global_clipnorm=1.0, state_bits=bits, fold_regularizers=True)  # noqa: E731
    nets = [_model(dev) for _ in range(3)]
    for net in nets:
        net(x, training=False)
    for net in nets[1:]:
        with torch.no_grad():
            for a, b in zip(net.parameters(), nets[0].parameters()):
                a.copy_(b)
    step = train_step_for(nets[0], x, y, optimizer=make, warmup=1)
    assert step.path == 'layers_graph'
    losses = [float(step()) for _ in range(4)]
    assert step.opt.iterations == 5
    for k, net in enumerate(nets[1:]):
        opt = make(net.parameters())
        for s in range(5):
            opt.zero_grad()
            loss = model_loss(net, ops.sparse_ce(net(x, training=True), y), True)
            (opt.backward(loss) if k == 0 else loss.backward())
            opt.step()
            if s:
                # the two ways add a bit-width's gradient pieces in another order: losses agree to fp32 rounding of the steps
                assert abs(float(loss) - losses[s - 1]) <= 1e-3 * abs(losses[s - 1])
    for a, b in zip(nets[0].parameters(), nets[1].parameters()):
        assert torch.isfinite(a).all() and float((a - b).abs().max()) <= 5 * 2 * 0.0021 + 1e-6  # (each step moves at most about lr)


def test_fit_with_adamw(dev):
    from hgq2_amd.train import AdamW, fit

    gen = torch.Generator().manual_seed(13)
    x, y = torch.randn(1000, 16, generator=gen).to(dev), torch.randint(0, 5, (1000,), generator=gen).to(dev)
    made = []

    def make(v):
        made.append(AdamW(v, lr=0.001, state_bits=8, fold_regularizers=True))
        return made[-1]

    hist = fit(_model(dev), x, y, batch_size=128, epochs=2, optimizer=make, seed=1)
    assert len(hist) == 2 and all(math.isfinite(h['loss']) for h in hist)
    assert len(made) == 1 and made[0].iterations == 16  # 8 batches an epoch, the last one shorter
    hist = fit(_model(dev), x, y, batch_size=500, epochs=1, lr=0.001, optimizer='adamw', seed=1)
    assert math.isfinite(hist[0]['loss'])


def test_what_the_class_refuses(dev):
    from hgq2_amd.train import AdamW

    p = torch.nn.Parameter(torch.ones(10, device=dev))
    with pytest.raises(ValueError, match='twice'):
        AdamW([p, p])
    with pytest.raises(ValueError, match='float32'):
        AdamW([torch.nn.Parameter(torch.ones(3, device=dev, dtype=torch.float64))])
    with pytest.raises(ValueError, match='one device'):
        AdamW([p, torch.nn.Parameter(torch.ones(3))])
    for data in (torch.ones(9, device=dev), torch.ones(10, device=dev, dtype=torch.bfloat16), torch.ones(10), torch.ones(20, device=dev)[::2]):
        q = torch.nn.Parameter(torch.ones(10, device=dev))
        opt = AdamW([q])
        q.data = data
        q.grad = torch.ones_like(q)
        before = q.detach().clone()
        with pytest.raises(ValueError, match='stay contiguous'):
            opt.step()
        assert torch.equal(q, before) and opt.iterations == 0
    q = torch.nn.Parameter(torch.ones(10, device=dev))
    opt = AdamW([q])
    q._hgq_side = [(None, torch.ones(9, device=dev))]
    with pytest.raises(ValueError, match='side gradient'):
        opt.step()
    with pytest.raises(AttributeError, match='32 bits'):
        opt.velocity_root
    with pytest.raises(AttributeError, match='8 bits'):
        AdamW([q], state_bits=8).velocity


def test_streams_and_a_sparse_gradient(dev):
    """Two optimizers that step on two streams at once do what they do one after the other; a sparse gradient is refused."""
    from hgq2_amd.train import AdamW

    gen = torch.Generator().manual_seed(14)
    data = [(torch.randn(200_000, generator=gen).to(dev), torch.randn(200_000, generator=gen).to(dev)) for _ in range(2)]

    def make():
        out = []
        for w, g in data:
            p = torch.nn.Parameter(w.clone())
            p.grad = g
            out.append((p, AdamW([p], global_clipnorm=1.0, state_bits=8, seed=2)))
        return out

    one, two = make(), make()
    for _ in range(4):
        for _, opt in one:
            opt.step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in two]
    for _ in range(4):
        for (_, opt), s in zip(two, streams):
            with torch.cuda.stream(s):
                opt.step()
    torch.cuda.synchronize()
    for (a, x), (b, y) in zip(one, two):
        assert torch.equal(a, b) and torch.equal(x.momentum.view(torch.uint8), y.momentum.view(torch.uint8)) and torch.equal(x.grad_norm, y.grad_norm)
    p = torch.nn.Parameter(torch.ones(4, 3, device=dev))
    opt = AdamW([p])
    p.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.ones(1, 3), (4, 3)).to(dev)
    with pytest.raises(ValueError, match='dense'):
        opt.step()


def test_memory_that_is_shared_and_decay_that_changes(dev):
    from hgq2_amd import ops
    from hgq2_amd.train import AdamW

    buf = torch.zeros(12, device=dev)
    with pytest.raises(ValueError, match='share memory'):
        AdamW([torch.nn.Parameter(buf[:8]), torch.nn.Parameter(buf[4:])])
    ws, state = [buf[:4], buf[4:]], ops.adamw_state(dev, 0.1)
    moments = [ops.adamw_moments(8, dev) for _ in ws]
    with pytest.raises(ValueError, match='moments share memory'):
        ops.adamw_update_multi_([buf[:8], torch.zeros(8, device=dev)], [torch.ones(8, device=dev)] * 2, [moments[0], moments[0]], state)
    assert not buf.any() and int(state[0]) == 0

    a, b = (torch.nn.Parameter(torch.ones(5, device=dev)) for _ in range(2))
    opt = AdamW([a, b], lr=0.5, weight_decay=0.25)
    opt.exclude_from_weight_decay([b])
    a.grad, b.grad = torch.zeros_like(a), torch.zeros_like(b)
    opt.step()  # gradients of zero: the decay alone moves
    assert torch.equal(a, torch.full_like(a, 0.875)) and torch.equal(b, torch.ones_like(b))
    opt.weight_decay = 0.5
    opt.step()
    assert torch.equal(a, torch.full_like(a, 0.875 * 0.75)) and torch.equal(b, torch.ones_like(b)) and opt.weight_decay == 0.5
    with pytest.raises(ValueError, match='negative'):
        opt.weight_decay = -0.1


def test_more_elements_than_32_bits_count(dev):
    """2^32 + 1077 elements: the first and the last ones against 64 bits, and the norm (all other gradients are zero)."""
    from hgq2_amd import ops

    n, edge = 2**32 + 1077, 1077 + 3 * BLOCK
    gen = torch.Generator().manual_seed(15)
    w, g = (torch.zeros(n, dtype=torch.bfloat16, device=dev) for _ in range(2))
    ends = (slice(0, edge), slice(n - edge, n))  # (both begin with a block)
    assert (n - edge) % BLOCK == 0
    for e in ends:
        w[e], g[e] = torch.randn(edge, generator=gen).to(dev), torch.randn(edge, generator=gen).to(dev)
    assert abs(float(ops.global_norm([g])) - math.sqrt(sum(float((g[e].double()**2).sum()) for e in ends))) <= 2 * U * 100
    moments, state = ops.adamw_moments(n, dev, 8), ops.adamw_state(dev, 0.001)
    before = [w[e].clone() for e in ends]
    ops.adamw_update_multi_([w], [g], [moments], state, decay=[0.004], seed=9)
    for e, old in zip(ends, before):
        zero = torch.zeros(edge)
        nw, nm, nv, tw, tm, tv = _plain(old, g[e], zero, zero, 1)
        _near(w[e], nw, tw, torch.bfloat16, 'w')
        h = _philox(np.arange(e.start // 4, -(-e.stop // 4), dtype=np.uint64), 1, 9)[:edge]
        scales = slice(e.start // BLOCK, -(-e.stop // BLOCK))
        _codes_near(moments[0][e], moments[1][scales], nm, tm, h & np.uint64(0xFFFF), False, 'm')
        r = nv.sqrt()
        _codes_near(moments[2][e], moments[3][scales], r, tv / (2 * r).clamp(min=1e-300) + 2 * U * r, h >> np.uint64(16), True, 'r')
    assert not w[edge:n - edge].any()


def test_fit_counts_regularizers_once(dev):
    """An epoch's loss is the same whether the optimizer folds the regularizers into its launch or they are terms of the loss."""
    from hgq2_amd.regularizers import MonoL1
    from hgq2_amd.train import AdamW, fit

    gen = torch.Generator().manual_seed(16)
    x, y = torch.randn(512, 16, generator=gen).to(dev), torch.randint(0, 5, (512,), generator=gen).to(dev)
    nets, losses = [_model(dev) for _ in range(2)], []
    for net in nets:
        net(x, training=False)
    with torch.no_grad():
        for a, b in zip(nets[1].parameters(), nets[0].parameters()):
            a.copy_(b)
    for fold, net in zip((True, False), nets):
        regularised = [p for p in net.parameters() if p.requires_grad and isinstance(getattr(p, 'regularizer', None), MonoL1)]
        assert regularised
        for p in regularised:
            p.regularizer = MonoL1(1e-4)
        hist = fit(net, x, y, batch_size=128, lr=0.0, shuffle=False,
                   optimizer=lambda v: AdamW(v, lr=0.0, weight_decay=0.0, fold_regularizers=fold))  # noqa: B023
        losses.append(hist[0]['loss'])
        total = sum(float(p.regularizer(p)) for p in regularised)
        assert total > 0.01
    assert abs(losses[0] - losses[1]) <= 1e-5 * abs(losses[0])


def test_gradients_that_are_views(dev):
    """Gradients that are lazily negated, expanded or transposed count as what they stand for."""
    from hgq2_amd import ops
    from hgq2_amd.train import AdamW

    gen = torch.Generator().manual_seed(18)
    base = torch.randn(6, 40, generator=gen).to(dev)
    views = [torch._neg_view(base), base[:1].expand(6, 40), base.t().contiguous().t(), torch.view_as_complex(base.view(6, 20, 2)).conj().imag.repeat(1, 2)]
    for g in views:
        a, b = (torch.nn.Parameter(torch.ones(6, 40, device=dev)) for _ in range(2))
        a.grad, b.grad = g, g.clone(memory_format=torch.contiguous_format).resolve_neg()
        one, two = AdamW([a], global_clipnorm=1.0), AdamW([b], global_clipnorm=1.0)
        one.step(), two.step()
        assert torch.equal(a, b) and torch.equal(one.momentum, two.momentum) and torch.equal(one.grad_norm, two.grad_norm)
        assert torch.equal(ops.global_norm([g]), one.grad_norm)
        c, state = torch.ones(6, 40, device=dev), ops.adamw_state(dev, 0.001)
        ops.adamw_update_multi_([c], [g], [ops.adamw_moments(240, dev)], state, decay=[0.004], clipnorm=1.0)
        assert torch.equal(c, a)
    p = torch.nn.Parameter(torch.ones(6, 40, device=dev))
    opt = AdamW([p])
    p.data = torch._neg_view(p.data)
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match='stay contiguous'):
        opt.step()


def test_recording_beside_a_living_loss_is_refused(dev):
    from hgq2_amd import ops
    from hgq2_amd.train import AdamW, model_loss, train_step_for

    gen = torch.Generator().manual_seed(20)
    x, y = torch.randn(128, 16, generator=gen).to(dev), torch.randint(0, 5, (128,), generator=gen).to(dev)
    net = _model(dev)
    net(x, training=False)
    opt = AdamW(net.parameters(), fold_regularizers=True)
    for _ in range(2):
        opt.zero_grad()
        loss = model_loss(net, ops.sparse_ce(net(x, training=True), y), True)
        opt.backward(loss)
        opt.step()
    with pytest.raises(RuntimeError, match='another stream that is still alive'):
        train_step_for(net, x, y, optimizer='adamw')
    del loss
    step = train_step_for(net, x, y, optimizer='adamw')
    assert math.isfinite(float(step())) and step.opt.iterations == 4
