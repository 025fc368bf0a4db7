"""The operators of a training step, as a user's program calls them: the cases
that are timed, their inputs, one pass in plain torch operations or through the
framework's entry points, the work a pass cannot do without, and its results in
64 bits.

A case names an operator:
  linear    y = act(x W^T + bias) + residual (``dir`` fwd), or the gradients of
            x, W and bias from that of y and the saved x W^T + bias (``dir`` bwd);
  loss      softmax cross-entropy of rows of logits and its gradient;
  adamw     one AdamW step over many tensors, states in 32 or in 8 bits.
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
TYPES = {'fp32': F32, 'bf16': BF16}

ACAS = '5-50-50-50-50-50-50-5'
BLOCK = 256      # values that share a scale, and what a tensor's state is padded to
E4M3_MAX = 448.0
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.1


def listed():
    return [
        # one token through a projection: the weights' bytes and a launch
        {'name': 'linear_token', 'op': 'linear', 'dir': 'fwd', 'type': 'bf16', 'M': 1, 'K': 4096,
         'N': 4096, 'act': 'silu', 'residual': False},
        # the 784-1024 layer of the MNIST-sized net on the batch that is verified
        {'name': 'linear_net', 'op': 'linear', 'dir': 'fwd', 'type': 'fp32', 'M': 512, 'K': 784,
         'N': 1024, 'act': 'relu', 'residual': False},
        # the wide half of a feed-forward block over many tokens
        {'name': 'linear_block', 'op': 'linear', 'dir': 'fwd', 'type': 'bf16', 'M': 8192,
         'K': 4096, 'N': 16384, 'act': 'gelu', 'residual': False},
        # backward of the 784-1024 layer over a training batch
        {'name': 'linear_bwd_net', 'op': 'linear', 'dir': 'bwd', 'type': 'fp32', 'M': 4096,
         'K': 784, 'N': 1024, 'act': 'relu'},
        # backward of a square layer over many tokens
        {'name': 'linear_bwd_block', 'op': 'linear', 'dir': 'bwd', 'type': 'bf16', 'M': 8192,
         'K': 4096, 'N': 4096, 'act': 'gelu'},
        # widths and a batch that fill no tile and align to no load
        {'name': 'linear_bwd_odd', 'op': 'linear', 'dir': 'bwd', 'type': 'bf16', 'M': 1021,
         'K': 333, 'N': 777, 'act': 'silu'},
        # ten classes: the verified nets' own loss, launches only
        {'name': 'loss_classes', 'op': 'loss', 'type': 'fp32', 'rows': 512, 'classes': 10,
         'ignored': 0.0, 'masked': 0, 'smoothing': 0.0},
        # a vocabulary of odd size in 32 bits, smoothed, a third of the rows padding
        {'name': 'loss_odd', 'op': 'loss', 'type': 'fp32', 'rows': 1000, 'classes': 50021,
         'ignored': 0.33, 'masked': 0, 'smoothing': 0.1},
        # a training batch's tokens over a large vocabulary padded to a round size
        {'name': 'loss_vocab', 'op': 'loss', 'type': 'bf16', 'rows': 8192, 'classes': 131072,
         'ignored': 0.05, 'masked': 200, 'smoothing': 0.0},
        # every tensor of the small net: a launch
        {'name': 'adamw_net', 'op': 'adamw', 'bits': 32, 'tensors': ACAS, 'param': 'fp32',
         'grad': 'fp32', 'copy': False},
        # 403 million parameters, gradients and working copies in bf16
        {'name': 'adamw_layers', 'op': 'adamw', 'bits': 32, 'tensors': '-'.join(
            ['2048', '8192'] * 12 + ['2048']), 'param': 'fp32', 'grad': 'bf16', 'copy': True},
        # many tensors of ragged sizes, states in 8 bits
        {'name': 'adamw_ragged', 'op': 'adamw', 'bits': 8, 'tensors': 'ragged-300-200000000',
         'param': 'fp32', 'grad': 'bf16', 'copy': True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges; sizes by their logarithm, odd
    ones as likely as even ones."""
    op = rng.choice(['linear', 'linear', 'linear', 'loss', 'adamw'])
    if op == 'linear':
        kind = rng.choice(['fp32', 'bf16'])
        most = 4e10 if kind == 'fp32' else 2.7e11
        while True:
            M, K, N = _log(rng, 1, 8192), _log(rng, 8, 16384), _log(rng, 8, 16384)
            if rng.random() < 0.5:  # half of them aligned, as most nets' widths are
                K, N = K + -K % 64, N + -N % 64
            if M * K * N <= most:
                break
        case = {'op': op, 'dir': rng.choice(['fwd', 'bwd']), 'type': kind, 'M': M, 'K': K, 'N': N,
                'act': rng.choice(['none', 'relu', 'gelu', 'silu'])}
        if case['dir'] == 'fwd':
            case['residual'] = rng.random() < 0.5
        return case
    if op == 'loss':
        kind, classes = rng.choice(['fp32', 'bf16']), _log(rng, 2, 131072)
        rows = _log(rng, 1, min(65536, int(5e8 / classes)))
        smooth = rng.choice([0.0, 0.1])
        return {'op': op, 'type': kind, 'rows': rows, 'classes': classes,
                'ignored': rng.choice([0.0, 0.2]), 'smoothing': smooth,
                'masked': 0 if smooth else rng.randint(0, classes // 3)}
    total = _log(rng, 1e4, 3e8)
    return {'op': op, 'bits': rng.choice([8, 32]), 'param': rng.choice(['fp32', 'fp32', 'bf16']),
            'tensors': 'ragged-%d-%d' % (rng.randint(1, 300), total),
            'grad': rng.choice(['fp32', 'bf16']), 'copy': rng.random() < 0.5}


# -------------------------------------------------------------------- inputs

def _sizes(case):
    """Values of each tensor of an optimiser step."""
    t = case['tensors'].split('-')
    if t[0] == 'ragged':
        r = random.Random(int(t[1]) * 1000003 + int(t[2]))
        w = [math.exp(r.gauss(0, 1.5)) for _ in range(int(t[1]))]
        return [max(1, int(int(t[2]) * x / sum(w))) for x in w]
    w = [int(v) for v in t]
    return [n for a, b in zip(w, w[1:]) for n in (a * b, b)]


def _padded(case):
    """Offset of each tensor in a buffer that pads each to whole blocks, and its length."""
    at, offs = 0, []
    for n in _sizes(case):
        offs.append(at)
        at += n + -n % BLOCK
    return offs, at


def prepare(case, seed):
    dev = torch.device('cuda:0')
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def randn(*shape, std=1.0, to=None):
        t = torch.randn(shape, generator=g, device=dev) * std
        return t if to is None else t.to(to)

    s = {'case': case}
    if case['op'] == 'linear':
        M, K, N, to = case['M'], case['K'], case['N'], TYPES[case['type']]
        s.update(x=randn(M, K, to=to), W=randn(N, K, std=K ** -0.5, to=to))
        if case['dir'] == 'fwd':
            s.update(b=randn(N, std=0.1, to=to), r=randn(M, N, to=to) if case['residual'] else None)
        else:
            s.update(dy=randn(M, N, std=M ** -0.5, to=to),
                     z=randn(M, N, to=to) if case['act'] != 'none' else None)
    elif case['op'] == 'loss':
        R, V = case['rows'], case['classes']
        s['logits'] = randn(R, V, std=3.0, to=TYPES[case['type']])
        if case['masked']:
            s['logits'][:, V - case['masked']:] = -math.inf
        t = torch.randint(0, V - case['masked'], (R,), generator=g, device=dev)
        skip = torch.rand(R, generator=g, device=dev) < case['ignored']
        skip[0] = False
        s['target'] = torch.where(skip, torch.full_like(t, -100), t)
    else:
        offs, n = _padded(case)
        sizes = _sizes(case)
        real = torch.zeros(n, dtype=torch.bool, device=dev)
        for o, k in zip(offs, sizes):
            real[o:o + k] = True
        # gradients of very different sizes side by side, some exactly zero
        mag = torch.exp(randn(n) * 1.5 - 8) * real
        flat = {'p': (randn(n, std=0.02) * real).to(TYPES[case['param']]),
                'g': (randn(n) * mag).to(TYPES[case['grad']]),
                'c': torch.zeros(n, dtype=BF16, device=dev) if case['copy'] else None}
        flat['g'][::97] = 0
        m, v = randn(n) * mag * 0.3, (mag * (0.5 + torch.rand(n, generator=g, device=dev))) ** 2
        if case['bits'] == 8:
            state = dict(zip(('m', 'm_scale'), _nearest(m)))
            state.update(zip(('v', 'v_scale'), _nearest(v.sqrt())))
        else:
            state = {'m': m, 'v': v}
        s.update(flat=flat, state=dict(state, bits=case['bits']), step=1000)
        s.update({k: [t[o:o + w] for o, w in zip(offs, sizes)] if t is not None else None
                  for k, t in flat.items()})
    return s


def _nearest(x):
    """Values as e4m3 bytes with a scale per block, to nearest: a state to begin with."""
    x = x.view(-1, BLOCK)
    scale = x.abs().amax(1, keepdim=True) / E4M3_MAX
    q = torch.where(scale > 0, x / scale, torch.zeros_like(x)).to(torch.float8_e4m3fn)
    return q.view(-1).view(torch.uint8), scale.view(-1).contiguous()


# ---------------------------------------------------------------- plain forms

def _act(z, name):
    if name == 'relu':
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == 'gelu':
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == 'silu':
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == 'relu':
        return (z > 0).to(z.dtype)
    if name == 'gelu':
        return (0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
                + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)))
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _plain_linear(s):
    c, to = s['case'], TYPES[s['case']['type']]
    x, W = s['x'].float(), s['W'].float()
    if c['dir'] == 'fwd':
        y = _act(x @ W.t() + s['b'].float(), c['act'])
        if s['r'] is not None:
            y = y + s['r'].float()
        return {'y': y.to(to)}
    dz = s['dy'].float()
    if s['z'] is not None:
        dz = dz * _slope(s['z'].float(), c['act'])
    return {'dx': (dz @ W).to(to), 'dW': (dz.t() @ x).to(to), 'db': dz.sum(0).to(to)}


def _plain_loss(s):
    c, t = s['case'], s['target']
    z, keep, e = s['logits'].float(), t >= 0, s['case']['smoothing']
    at = torch.where(keep, t, torch.zeros_like(t)).unsqueeze(1)
    m = z.amax(1, keepdim=True)
    p = torch.exp(z - m)
    total = p.sum(1, keepdim=True)
    lse = m + torch.log(total)
    loss = lse - (1 - e) * z.gather(1, at)
    if e:
        loss = loss - e * z.mean(1, keepdim=True)
    w = keep.float().unsqueeze(1) / keep.sum()
    p = p / total - e / c['classes']
    p.scatter_add_(1, at, torch.full_like(lse, e - 1))
    return {'loss': torch.where(keep.unsqueeze(1), loss, torch.zeros_like(loss)).sum() / keep.sum(),
            'dlogits': (p * w).to(s['logits'].dtype)}


def _dither(n, step, device):
    """20 bits for each value's rounding, from its place in the state and the step."""
    i = torch.arange(n, dtype=torch.int64, device=device)
    h = (i * 0x9E3779B9 + step * 0x6A09E667) & 0xffffffff
    h = ((h ^ (h >> 15)) * 0xBB67AE85) & 0xffffffff
    return ((h ^ (h >> 15)) >> 12).to(torch.int32)


def _encode(x, r, positive):
    """x as e4m3 bytes with a scale per block, rounded up with the probability of what is cut:
    values from the smallest normal up on the bits of the float, smaller ones on the
    fixed-point grid of the subnormals.  A positive value is never stored as zero."""
    x, r = x.view(-1, BLOCK), r.view(-1, BLOCK)
    top = x.abs().amax(1, keepdim=True)
    inv = torch.where(top >= 2.0 ** -100, E4M3_MAX / top, torch.zeros_like(top))
    scale = torch.where(top >= 2.0 ** -100, top * (1 / E4M3_MAX), torch.zeros_like(top))
    t = x.abs() * inv
    code = ((t.view(torch.int32) + r) >> 20) - 960
    small = (t * 512.0 + r.float() * 2.0 ** -20).to(torch.int32)
    code = torch.where(t < 2.0 ** -6, small, code).clamp(max=126)
    if positive:
        code = torch.where(t > 0, code.clamp(min=1), code)
    code = torch.where(x < 0, code + 128, code)
    return code.to(torch.uint8).view(-1), scale.view(-1)


def _decode(code, scale):
    return (code.view(torch.float8_e4m3fn).float().view(-1, BLOCK) * scale.unsqueeze(1)).view(-1)


def _outputs(s):
    f, st = s['flat'], s['state']
    out = {'p': f['p'], 'copy': f['c']}
    if st['bits'] == 8:
        return dict(out, m=st['m'].view(torch.float8_e4m3fn), m_scale=st['m_scale'],
                    v=st['v'].view(torch.float8_e4m3fn), v_scale=st['v_scale'])
    return dict(out, m=st['m'], v=st['v'])


def _plain_adamw(s):
    f, st, k = s['flat'], s['state'], s['step']
    b1, b2 = BETAS
    g, eight = f['g'].float(), st['bits'] == 8
    m = _decode(st['m'], st['m_scale']) if eight else st['m']
    v = _decode(st['v'], st['v_scale']).square() if eight else st['v']
    m = m * b1 + (1 - b1) * g
    v = v * b2 + (1 - b2) * g * g
    u = v.sqrt()
    p = f['p'].float() * (1 - LR * DECAY)
    p = p - LR / (1 - b1 ** k) * (m / (u / math.sqrt(1 - b2 ** k) + EPS))
    f['p'].copy_(p)
    if f['c'] is not None:
        f['c'].copy_(p)
    if eight:
        r = _dither(m.numel(), k, m.device)
        for x, key in ((m, 'm'), (u, 'v')):
            code, scale = _encode(x, r, key == 'v')
            st[key].copy_(code)
            st[key + '_scale'].copy_(scale)
    else:
        st['m'].copy_(m)
        st['v'].copy_(v)
    return _outputs(s)


# ---------------------------------------------------------------- one pass

def _train():
    at = os.path.join(_ROOT, 'vibecheck-nn_amd')
    if at not in sys.path:
        sys.path.insert(1, at)
    from vibecheck_amd import train
    return train


def run(s):
    c = s['case']
    if not own:
        return {'linear': _plain_linear, 'loss': _plain_loss, 'adamw': _plain_adamw}[c['op']](s)
    train = _train()
    if c['op'] == 'linear':
        act = None if c['act'] == 'none' else c['act']
        if c['dir'] == 'fwd':
            return {'y': train.linear(s['x'], s['W'], s['b'], act=act, residual=s['r'])}
        dx, dW, db = train.linear_backward(s['dy'], s['x'], s['W'], z=s['z'], act=act)
        return {'dx': dx, 'dW': dW, 'db': db}
    if c['op'] == 'loss':
        loss, dlogits = train.cross_entropy(s['logits'], s['target'], ignore_index=-100,
                                            smoothing=c['smoothing'])
        return {'loss': loss, 'dlogits': dlogits}
    train.adamw_step(s['p'], s['g'], s['state'], s['step'], lr=LR, betas=BETAS, eps=EPS,
                     weight_decay=DECAY, copies=s['c'])
    return _outputs(s)


def work(case):
    if case['op'] == 'linear':
        M, K, N, e = case['M'], case['K'], case['N'], 4 if case['type'] == 'fp32' else 2
        if case['dir'] == 'fwd':
            return {'bytes': e * (M * K + N * K + N + M * N * (2 if case['residual'] else 1)),
                    'flops': 2 * M * N * K}
        return {'bytes': e * (2 * M * K + 2 * N * K + N + M * N * (1 if case['act'] == 'none' else 2)),
                'flops': 4 * M * N * K}
    if case['op'] == 'loss':
        R, V, e = case['rows'], case['classes'], 4 if case['type'] == 'fp32' else 2
        return {'bytes': 2 * e * R * V + 8 * R + 4, 'flops': 8 * R * V}
    n = sum(_sizes(case))
    e = {'fp32': 4, 'bf16': 2}
    state = 16 if case['bits'] == 32 else 4 + 16 / BLOCK
    return {'bytes': n * (2 * e[case['param']] + e[case['grad']] + state + (2 if case['copy'] else 0)),
            'flops': 15 * n}


# ---------------------------------------------------------------- in 64 bits

def _exact_linear(s):
    c = s['case']
    x, W = s['x'].double(), s['W'].double()

    def phi(z):
        return torch.special.ndtr(z)

    if c['dir'] == 'fwd':
        z = torch.addmm(s['b'].double(), x, W.t())
        if c['act'] == 'relu':
            z = z.clamp(min=0)
        elif c['act'] == 'gelu':
            z = z * phi(z)
        elif c['act'] == 'silu':
            z = z * torch.sigmoid(z)
        return {'y': z if s['r'] is None else z + s['r'].double()}
    dz = s['dy'].double()
    if s['z'] is not None:
        z = s['z'].double()
        if c['act'] == 'relu':
            dz = torch.where(z > 0, dz, 0.0)
        elif c['act'] == 'gelu':
            dz = dz * (phi(z) + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi))
        else:
            q = torch.sigmoid(z)
            dz = dz * (q + z * q * torch.sigmoid(-z))
    return {'dx': torch.mm(dz, W), 'dW': torch.mm(dz.t(), x), 'db': dz.sum(0)}


def _exact_loss(s):
    e, t, V = s['case']['smoothing'], s['target'], s['case']['classes']
    z, keep = s['logits'].double(), s['target'] >= 0
    n, row = int(keep.sum()), torch.arange(t.numel(), device=t.device)[keep]
    q = torch.log_softmax(z, 1)
    loss = -(1 - e) * q[row, t[row]].sum() / n
    if e:
        loss = loss - e * q[row].mean(1).sum() / n
    grad = q.exp_() - e / V
    grad[row, t[row]] -= 1 - e
    grad *= (keep.double() / n).unsqueeze(1)
    return {'loss': loss, 'dlogits': grad}


def _exact_state(x, step, floor):
    """e4m3 values in units of the block's scale, and the scales: a value goes to the upper of
    its two neighbours on the grid where the part above the lower one, and a number in [0, 1)
    made of the value's place and the step, reach one."""
    h = torch.arange(x.numel(), device=x.device) * 0x9E3779B9 + step * 0x6A09E667
    h = h % 2 ** 32
    h = torch.bitwise_xor(h, h // 2 ** 15) * 0xBB67AE85 % 2 ** 32
    d = (torch.bitwise_xor(h, h // 2 ** 15) // 2 ** 12).double() / 2 ** 20
    del h
    x, d = x.reshape(-1, BLOCK), d.reshape(-1, BLOCK)
    scale = x.abs().amax(1, keepdim=True) / E4M3_MAX
    scale = torch.where(scale * E4M3_MAX >= 2.0 ** -100, scale, torch.zeros_like(scale))
    t = torch.where(scale > 0, x.abs() / scale, torch.zeros_like(x))
    grid = torch.exp2(torch.floor(torch.log2(t.clamp(min=2.0 ** -6))) - 3)
    q = (torch.floor(t / grid + d) * grid).clamp(max=E4M3_MAX)
    if floor:
        q = torch.where(t > 0, q.clamp(min=2.0 ** -9), q)
    return (q * torch.sign(x)).reshape(-1), scale.reshape(-1)


def _exact_adamw(s):
    f, st, k, (b1, b2) = s['flat'], s['state'], s['step'], BETAS
    g, m, v = f['g'].double(), st['m'], st['v']
    if st['bits'] == 8:
        m, v = (c.view(torch.float8_e4m3fn).float().double().reshape(-1, BLOCK)
                * st[key].double().reshape(-1, 1)
                for c, key in ((m, 'm_scale'), (v, 'v_scale')))
        m, v = m.reshape(-1), v.square().reshape(-1)
    m = torch.lerp(g, m.double(), b1)
    v = torch.lerp(g.square(), v.double(), b2)
    p = f['p'].double()
    p = p - LR * DECAY * p - LR * (m / (1 - b1 ** k)) / (torch.sqrt(v / (1 - b2 ** k)) + EPS)
    out = {'p': p, 'copy': None if f['c'] is None else p}
    if st['bits'] == 32:
        return dict(out, m=m, v=v)
    out['m'], out['m_scale'] = _exact_state(m, k, False)
    out['v'], out['v_scale'] = _exact_state(v.sqrt(), k, True)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {'linear': _exact_linear, 'loss': _exact_loss, 'adamw': _exact_adamw}[case['op']](s)
