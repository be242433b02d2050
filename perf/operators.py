"""The operators of an adaptive training step and of group-normalised layers, as cases that can be timed and compared.

* ``adamw``  - one AdamW step over all variables of a network (a kernel, a bias and their bit-width variables per layer),
  with both moments in 32 bits or in 8 bits with one scale per 256 elements, with or without clipping by the global norm.
* ``norm``   - the global norm of a network's gradients by itself (a monitor, or a clipping of the user's own).
* ``group``  - group normalisation with an activation over channels-last tensors: forward, or forward and backward.

Variables, gradients and moments of a network lie in one buffer each, every variable at a multiple of 256 elements; what
lies between them is zero and stays zero.

One AdamW step t = 1, 2, ... with a gradient g, element by element (the moments start at zero):

    g <- g min(1, clipnorm / norm(all g))                  (with clipping)
    m <- m + (g - m) (1 - beta_1);   v <- v + (g g - v) (1 - beta_2)
    w <- w - w (lr weight_decay)
    w <- w - m alpha / (sqrt(v) + epsilon),   alpha = lr sqrt(1 - beta_2^t) / (1 - beta_1^t)

With moments in 8 bits, m and r = sqrt(v) are held as E4M3 codes times a power of two s per block of 256 elements, which
brings the block's largest magnitude into [128, 256).  |x| / s is rounded stochastically: with u the spacing of E4M3 at
|x| / s, the code's value is u floor(|x| / (s u) + h / 2^16).  The 16-bit numbers h of element e are the halves (low: m, high: r)
of word e % 4 of Philox4x32-7 with counter (e / 4, t) and key seed.  An r that is not zero is held as at least the
smallest code, so that a step is never divided by epsilon alone.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 256
LR, WEIGHT_DECAY, BETA_1, BETA_2, EPSILON = 3e-4, 0.004, 0.9, 0.999, 1e-7
STEP = 1000  # steps before the one that is measured
GROUP_EPSILON = 1e-3

_TYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


def listed():
    return [
        # the benchmark's jet classifier: 28 variables of a few thousand elements, nothing but latency
        dict(name='adamw_mlp', op='adamw', dims='16-64-32-32-5', bits=32, clip=0.0, dtype='float32'),
        # a wide classifier, gradients clipped by their global norm
        dict(name='adamw_wide_clip', op='adamw', dims='256-512-256-128-10', bits=32, clip=0.5, dtype='float32'),
        # large layers with a bit-width of its own for every weight: three variables per weight, 150 million elements
        dict(name='adamw_large_clip', op='adamw', dims='4096-4096-4096-4096', bits=32, clip=1.0, dtype='float32'),
        # 16-bit variables and gradients of odd widths beside moments in 32 bits
        dict(name='adamw_bf16_odd', op='adamw', dims='2047-4001-1021', bits=32, clip=0.0, dtype='bfloat16'),
        # moments in 8 bits, the wide classifier
        dict(name='adamw8_wide', op='adamw', dims='256-512-256-128-10', bits=8, clip=0.5, dtype='float32'),
        # moments in 8 bits, large layers: what they are for
        dict(name='adamw8_large', op='adamw', dims='4096-4096-4096-4096', bits=8, clip=0.0, dtype='float32'),
        # the gradients' norm of the wide classifier, watched every step
        dict(name='norm_wide', op='norm', dims='256-512-256-128-10', dtype='float32'),
        # the same of large layers with odd widths in 16 bits
        dict(name='norm_large_odd', op='norm', dims='4001-4095-4001', dtype='bfloat16'),
        # one image through one layer of a trained network: nothing but latency
        dict(name='group_one_image', op='group', batch=1, height=28, width=28, channels=32, groups=8, act='relu', train=False, dtype='float32'),
        # the benchmark's image network, normalised per sample behind its first convolution, in training
        dict(name='group_conv_train', op='group', batch=1024, height=26, width=26, channels=32, groups=8, act='relu', train=True, dtype='float32'),
        # jets of 30 particles with an odd number of them per batch: short rows, many samples
        dict(name='group_particles_train', op='group', batch=1531, height=1, width=30, channels=48, groups=6, act='linear', train=True, dtype='float32'),
        # wide feature maps in 16 bits, forward and backward: the largest
        dict(name='group_maps_train_bf16', op='group', batch=48, height=64, width=64, channels=512, groups=32, act='silu', train=True, dtype='bfloat16'),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(['adamw', 'adamw', 'adamw', 'norm', 'group', 'group', 'group'])
    dtype = rng.choice(['float32', 'float32', 'bfloat16', 'float16'])
    if op == 'group':
        groups = _log(rng, 1, 32)
        channels = groups * _log(rng, 1, 24)
        height, width = rng.choice([(1, _log(rng, 1, 200)), (_log(rng, 2, 80), _log(rng, 2, 80))])
        most = max(1, min(2000, 100_000_000 // (channels * height * width)))
        return dict(op=op, batch=_log(rng, 1, most), height=height, width=width, channels=channels, groups=groups,
                    act=rng.choice(['linear', 'relu', 'silu']), train=rng.random() < 0.7, dtype=dtype)
    dims = '-'.join(str(_log(rng, 3, 2500)) for _ in range(rng.randint(2, 6)))
    if op == 'norm':
        return dict(op=op, dims=dims, dtype=dtype)
    return dict(op=op, dims=dims, bits=rng.choice([8, 32]), clip=rng.choice([0.0, 0.1, 1.0]), dtype=dtype)


def _sizes(case):
    """Elements of each variable of a stack of dense layers whose weights have bit-widths of their own."""
    dims = [int(d) for d in case['dims'].split('-')]
    sizes = []
    for k, n in zip(dims, dims[1:]):
        sizes += [k * n] * 3 + [n] * 3 + [k]  # kernel, its b and i; bias, its b and i; f of the inputs
    return sizes


def _layout(sizes):
    """Where each variable begins, and the length of the buffer."""
    at, n = [], 0
    for s in sizes:
        at.append(n)
        n += -(-s // BLOCK) * BLOCK
    return at, n


# ---- moments in 8 bits: plain arithmetic on whole numbers and floats -------------------------------------------------
def _philox(blocks, step, seed):
    """Four 32-bit words (in int64) per counter (block, step) under the key seed: Philox4x32 with seven rounds."""
    mask = 0xFFFFFFFF
    c0, c1 = blocks & mask, blocks >> 32
    c2, c3 = torch.full_like(blocks, step & mask), torch.full_like(blocks, step >> 32)
    k0, k1 = seed & mask, (seed >> 32) & mask
    for _ in range(7):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # (the low 64 bits of the product, as a signed number)
        c0, c1, c2, c3 = ((p1 >> 32) & mask) ^ c1 ^ k0, p1 & mask, ((p0 >> 32) & mask) ^ c3 ^ k1, p0 & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)


def _pow2(n):
    return ((n.to(torch.int32) + 127) << 23).view(torch.float32)


def _encode(x, h, floor):
    """E4M3 codes and scales of x (a whole number of blocks) with the 16-bit numbers h; `floor`: not zero stays not zero."""
    a = x.abs().reshape(-1, BLOCK)
    most = a.amax(dim=1)
    top = torch.where(most > 0, torch.frexp(most)[1], -118).clamp(min=-118)  # the largest lies in [2^(top - 1), 2^top)
    a = a * _pow2(8 - top)[:, None]
    unit = torch.frexp(a)[1].clamp(min=-5) - 4  # the exponent of the spacing: 3 bits behind the first, 2^-9 at the least
    q = torch.floor(a * _pow2(-unit) + h.reshape(a.shape).to(a.dtype) / 65536)
    y = q * _pow2(unit)
    if floor:
        y = torch.where((a > 0) & (y == 0), torch.full_like(y, 2.0**-9), y)
    y = torch.copysign(y, x.reshape(-1, BLOCK)).reshape(-1)
    return y.float().to(torch.float8_e4m3fn), (top + 119).to(torch.uint8).view(torch.float8_e8m0fnu)


def _decode(codes, scales):
    return (codes.float().reshape(-1, BLOCK) * scales.float()[:, None]).reshape(-1)


# ---- states ----------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = _TYPES[case['dtype']]
    state = {'case': case, 'seed': seed}
    if case['op'] == 'group':
        shape = (case['batch'], case['height'], case['width'], case['channels'])
        C = case['channels']
        x = torch.randn(shape, generator=g, device=dev)
        x.mul_(0.3 + torch.rand(C, generator=g, device=dev)).add_(torch.randn(C, generator=g, device=dev))
        state['x'] = x.to(dtype).requires_grad_(case['train'])
        state['gamma'] = (1 + 0.2 * torch.randn(C, generator=g, device=dev)).requires_grad_(case['train'])
        state['beta'] = (0.2 * torch.randn(C, generator=g, device=dev)).requires_grad_(case['train'])
        state['dy'] = torch.randn(shape, generator=g, device=dev).to(dtype) if case['train'] else None
        return state
    sizes = _sizes(case)
    at, n = _layout(sizes)
    spread = torch.exp(torch.randn(len(sizes), generator=g, device=dev).mul_(0.7)).mul_(1e-3)  # gradients of each variable
    inside = torch.zeros(n, device=dev)
    for a, s, k in zip(at, sizes, spread.unbind()):
        inside[a:a + s] = k
    state['grads'] = torch.randn(n, generator=g, device=dev).mul_(inside).to(dtype)
    views = list(zip(at, sizes))
    if case['op'] == 'norm':
        state['views'] = [state['grads'][a:a + s] for a, s in views]
        return state
    weights = torch.randn(n, generator=g, device=dev).mul_(0.05).mul_(inside > 0).to(dtype)
    m = torch.randn(n, generator=g, device=dev).mul_(0.25).mul_(inside)
    v = torch.rand(n, generator=g, device=dev).add_(0.5).mul_(inside).mul_(inside)
    state.update(weights=weights, step=STEP)
    if case['bits'] == 32:
        state['moments'] = [m, v]
    else:
        words = torch.randint(0, 2**16, (2, n), generator=g, device=dev)
        state['moments'] = [*_encode(m, words[0], False), *_encode(torch.sqrt(v), words[1], True)]
    state['views'] = views
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if own and case['op'] == 'adamw':
        from hgq2_amd.train import AdamW

        params = [torch.nn.Parameter(state['weights'][a:a + s]) for a, s in state['views']]
        for p, (a, s) in zip(params, state['views']):
            p.grad = state['grads'][a:a + s]
        opt = AdamW(params, lr=LR, weight_decay=WEIGHT_DECAY, beta_1=BETA_1, beta_2=BETA_2, epsilon=EPSILON,
                    global_clipnorm=case['clip'] or None, state_bits=case['bits'], seed=seed)
        names = ('momentum', 'velocity') if case['bits'] == 32 else ('momentum', 'momentum_scale', 'velocity_root', 'velocity_scale')
        opt.load_state_dict({'iterations': STEP, **dict(zip(names, state['moments']))})
        state['opt'], state['moments'] = opt, [getattr(opt, k) for k in names]
    return state


# ---- plain forms -----------------------------------------------------------------------------------------------------
def _adamw(s):
    case = s['case']
    s['step'] += 1
    t = s['step']
    alpha = LR * math.sqrt(1 - BETA_2**t) / (1 - BETA_1**t)
    g = s['grads'].float()
    if case['clip']:
        norm = torch.sqrt(torch.sum(g.double() ** 2)).float()
        g = g * torch.clamp(case['clip'] / norm, max=1.0)
    if case['bits'] == 32:
        m, v = s['moments']
    else:
        m = _decode(*s['moments'][:2])
        v = _decode(*s['moments'][2:]) ** 2
    m = m + (g - m) * (1 - BETA_1)
    v = v + (g * g - v) * (1 - BETA_2)
    r = torch.sqrt(v)
    w = s['weights'].float()
    w = w - w * (LR * WEIGHT_DECAY)
    w = w - m * alpha / (r + EPSILON)
    s['weights'].copy_(w)
    if case['bits'] == 32:
        for old, new in zip(s['moments'], (m, v)):
            old.copy_(new)
    else:
        words = _philox(torch.arange(m.numel() // 4, device=m.device), t, s['seed'])
        s['moments'] = [*_encode(m, words & 0xFFFF, False), *_encode(r, words >> 16, True)]
    return [s['weights'], *s['moments']]


def _activate(z, act):
    return torch.clamp(z, min=0) if act == 'relu' else z * torch.sigmoid(z) if act == 'silu' else z


def _group(s):
    case = s['case']
    G = case['groups']
    x = s['x'].detach().float()
    by = x.reshape(x.shape[0], -1, G, x.shape[-1] // G)  # batch, positions, groups, channels of a group
    mean = by.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((by - mean) ** 2).mean(dim=(1, 3), keepdim=True) + GROUP_EPSILON)
    xhat = ((by - mean) * rstd).reshape(x.shape)
    gamma = s['gamma'].detach()
    z = xhat * gamma + s['beta'].detach()
    y = _activate(z, case['act']).to(s['x'].dtype)
    if not case['train']:
        return [y]
    dz = s['dy'].float()
    if case['act'] == 'relu':
        dz = dz * (z > 0)
    elif case['act'] == 'silu':
        p = torch.sigmoid(z)
        dz = dz * (p * (1 + z * (1 - p)))
    dgamma, dbeta = (dz * xhat).sum(dim=(0, 1, 2)), dz.sum(dim=(0, 1, 2))
    d = (dz * gamma).reshape(by.shape)
    h = xhat.reshape(by.shape)
    dx = (d - d.mean(dim=(1, 3), keepdim=True) - h * (d * h).mean(dim=(1, 3), keepdim=True)) * rstd
    return [y, dx.reshape(x.shape).to(s['x'].dtype), dgamma, dbeta]


def run(state):
    case = state['case']
    if own:
        if case['op'] == 'adamw':
            state['opt'].step()
            return [state['weights'], *state['moments']]
        from hgq2_amd import ops

        if case['op'] == 'norm':
            return [ops.global_norm(state['views'])]
        x, gamma, beta = state['x'], state['gamma'], state['beta']
        if not case['train']:
            with torch.no_grad():
                return [ops.group_norm(x, case['groups'], gamma, beta, GROUP_EPSILON, case['act'])]
        y = ops.group_norm(x, case['groups'], gamma, beta, GROUP_EPSILON, case['act'])
        return [y.detach(), *torch.autograd.grad(y, [x, gamma, beta], state['dy'])]
    if case['op'] == 'adamw':
        return _adamw(state)
    if case['op'] == 'norm':
        return [torch.sqrt(torch.sum(state['grads'].float().double() ** 2)).float()]
    return _group(state)


def work(case):
    size = 4 if case['dtype'] == 'float32' else 2
    if case['op'] == 'group':
        n = case['batch'] * case['height'] * case['width'] * case['channels']
        return dict(bytes=n * size * (4 if case['train'] else 2), flops=n * (25 if case['train'] else 8))  # x, y (and dy, dx)
    n = sum(_sizes(case))
    if case['op'] == 'norm':
        return dict(bytes=n * size, flops=2 * n)
    moments = 16 * n if case['bits'] == 32 else 4 * n + 4 * (n // BLOCK)
    return dict(bytes=n * size * 3 + moments, flops=n * (16 if case['bits'] == 32 else 80))


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def _exact_codes(x, bits, keep):
    """Values of the codes and of the scales, by the distance of neighbouring E4M3 numbers: x in 64 bits, bits = h / 2^16."""
    rows = x.view(-1, BLOCK)
    most = rows.abs().max(dim=1, keepdim=True).values
    e = torch.floor(torch.log2(most.clamp(min=2.0**-119)))
    e = torch.where(torch.exp2(e) > most, e - 1, e)  # (a logarithm that was rounded up to a whole number)
    e = torch.where(torch.exp2(e + 1) <= most, e + 1, e).clamp(min=-119)
    scale = torch.exp2(e - 7)
    q = rows.abs() / scale
    d = torch.full_like(q, 2.0**-9)
    for k in range(-5, 9):  # binades of E4M3: [2^k, 2^(k + 1)) has steps of 2^(k - 3)
        d = torch.where(q >= 2.0**k, torch.full_like(q, 2.0 ** (k - 3)), d)
    y = torch.floor(q / d + bits.view(-1, BLOCK)) * d
    if keep:
        y = torch.where(q > 0, y.clamp(min=2.0**-9), y)
    return (y * torch.sign(rows)).view(-1), scale.view(-1)


def exact(case, seed):
    s = _inputs(case, seed)
    if case['op'] == 'norm':
        return [torch.linalg.vector_norm(s['grads'].double())]
    if case['op'] == 'group':
        x = s['x'].detach().double().requires_grad_(case['train'])
        gamma, beta = (s[k].detach().double().requires_grad_(case['train']) for k in ('gamma', 'beta'))
        B, C, G = x.shape[0], x.shape[-1], case['groups']
        g = x.movedim(-1, 1).reshape(B, G, -1)
        var, mean = torch.var_mean(g, dim=2, correction=0, keepdim=True)
        z = ((g - mean) / (var + GROUP_EPSILON).sqrt()).reshape(B, C, *x.shape[1:-1]).movedim(1, -1) * gamma + beta
        y = z.relu() if case['act'] == 'relu' else z / (1 + torch.exp(-z)) if case['act'] == 'silu' else z
        if not case['train']:
            return [y]
        return [y.detach(), *torch.autograd.grad(y, [x, gamma, beta], s['dy'].double())]
    t = STEP + 1
    g = s['grads'].double()
    if case['clip']:
        g = g * min(1.0, case['clip'] / float(torch.linalg.vector_norm(g)))
    if case['bits'] == 32:
        m, v = (k.double() for k in s['moments'])
    else:
        codes = [k.double() for k in s['moments']]
        m, v = ((c.view(-1, BLOCK) * q.view(-1, 1)).view(-1) for c, q in (codes[:2], codes[2:]))
        v = v.square()
    m = BETA_1 * m + (1 - BETA_1) * g
    v = BETA_2 * v + (1 - BETA_2) * g.square()
    w = s['weights'].double() * (1 - LR * WEIGHT_DECAY)
    w = w - (LR * math.sqrt(-math.expm1(t * math.log(BETA_2))) / -math.expm1(t * math.log(BETA_1))) * m / (v.sqrt() + EPSILON)
    if case['bits'] == 32:
        return [w, m, v]
    h = _philox(torch.arange(m.numel() // 4, device=m.device), t, s['seed'])  # (whole numbers: there is one way only)
    return [w, *_exact_codes(m, (h % 65536).double() / 65536, False), *_exact_codes(v.sqrt(), (h // 65536).double() / 65536, True)]
