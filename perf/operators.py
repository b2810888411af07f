"""What the sequence-block operators are timed and checked on: layer norm, the short causal convolution and the
selective scan, each for training (forward and backward in one pass), for prompts and for single tokens.

A case says which operator, its type and its sizes.  `run` makes one pass: with `own` false in plain torch operations
in 32 bits, with `own` true through ps_vae_amd.ops.  `exact` computes the same outputs from the definitions in 64
bits, step by step along every sequence.

  layer norm   y = (x - mean) * rstd * w + b over the last dimension
  convolution  y[t, d] = silu(b[d] + sum_k w[d, k] x[t - W + 1 + k, d]), rows of other sequences read as zero
  scan         delta = softplus(dt + dt_bias);  h[t] = exp(delta A) h[t-1] + delta x[t] B[t];
               y[t] = (sum_n C[t, n] h[t, n] + D x[t]) * silu(z[t])
"""
import math
import random

import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}
EPS = 1e-5


def listed():
    return [
        # the norm in front of a block while a handful of sequences is decoded: latency
        {'name': 'norm 4 x 300 f32', 'op': 'norm', 'type': 'f32', 'rows': 4, 'width': 300, 'grad': False},
        # a training batch of the molecule decoder: 128 graphs of about 25 pieces, the hidden width of the encoder
        {'name': 'norm 3277 x 300 f32 train', 'op': 'norm', 'type': 'f32', 'rows': 3277, 'width': 300, 'grad': True},
        # a training batch of long sequences at a generic width
        {'name': 'norm 32768 x 2048 bf16 train', 'op': 'norm', 'type': 'bf16', 'rows': 32768, 'width': 2048, 'grad': True},
        # the convolution's token step for a serving batch
        {'name': 'conv step 64 x 4096 bf16', 'op': 'conv_step', 'type': 'bf16', 'seqs': 64, 'width': 4096, 'taps': 4},
        # ragged piece sequences of a training batch, no sequence longer than the 50 positions of the model's table
        {'name': 'conv 128 ragged x 600 f32 train', 'op': 'conv', 'type': 'f32', 'seqs': 128, 'longest': 50, 'ragged': True,
         'width': 600, 'taps': 4, 'grad': True},
        # a training batch of long sequences
        {'name': 'conv 8 x 2048 x 2048 bf16 train', 'op': 'conv', 'type': 'bf16', 'seqs': 8, 'longest': 2048, 'ragged': False,
         'width': 2048, 'taps': 4, 'grad': True},
        # one molecule decoded token by token: latency
        {'name': 'scan step 1 x 600 f32', 'op': 'scan_step', 'type': 'f32', 'seqs': 1, 'width': 600, 'states': 16, 'groups': 1},
        # a full serving batch: bound by the states' memory traffic
        {'name': 'scan step 256 x 4096 bf16', 'op': 'scan_step', 'type': 'bf16', 'seqs': 256, 'width': 4096, 'states': 16, 'groups': 1},
        # ragged piece sequences of a training batch, the initial state made from the latents
        {'name': 'scan 128 ragged x 600 f32 train', 'op': 'scan', 'type': 'f32', 'seqs': 128, 'longest': 50, 'ragged': True,
         'width': 600, 'states': 16, 'groups': 1, 'grad': True},
        # one long prompt of an odd length: nothing but the time axis to spread over the chip
        {'name': 'scan 1 x 8191 x 2048 bf16 prompt', 'op': 'scan', 'type': 'bf16', 'seqs': 1, 'longest': 8191, 'ragged': False,
         'width': 2048, 'states': 16, 'groups': 1, 'grad': False},
        # a training batch of long sequences
        {'name': 'scan 8 x 2048 x 2048 bf16 train', 'op': 'scan', 'type': 'bf16', 'seqs': 8, 'longest': 2048, 'ragged': False,
         'width': 2048, 'states': 16, 'groups': 1, 'grad': True},
        # many states a channel, several groups of B and C, ragged lengths, an odd width
        {'name': 'scan 5 ragged x 1004 f16 64 states train', 'op': 'scan', 'type': 'f16', 'seqs': 5, 'longest': 1500, 'ragged': True,
         'width': 1004, 'states': 64, 'groups': 4, 'grad': True},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(['norm', 'norm', 'conv_step', 'conv', 'scan_step', 'scan', 'scan', 'scan'])
    kind = rng.choice(['f32', 'bf16', 'f16'])
    if op == 'norm':
        width = _log_int(rng, 8, 16384)
        rows = _log_int(rng, 1, min(40000, 32768 * 2048 // width // (BYTES[kind] // 2)))
        return {'op': op, 'type': kind, 'rows': rows, 'width': width, 'grad': rng.random() < 0.7}
    if op == 'conv_step':
        return {'op': op, 'type': kind, 'seqs': _log_int(rng, 1, 512), 'width': _log_int(rng, 8, 8192), 'taps': rng.randint(1, 8)}
    if op == 'scan_step':
        groups = rng.choice([1, 1, 2, 4])
        return {'op': op, 'type': kind, 'seqs': _log_int(rng, 1, 256), 'width': groups * _log_int(rng, 8, 4096 // groups),
                'states': rng.choice([1, 5, 8, 16, 16]), 'groups': groups}
    groups = rng.choice([1, 1, 2, 4]) if op == 'scan' else 1
    states = rng.choice([1, 4, 7, 8, 16, 16, 32, 64]) if op == 'scan' else 1
    width = groups * _log_int(rng, 8, 2048 // groups)
    rows = 8 * 2048 * 2048 // width // max(1, states // 16) // (BYTES[kind] // 2)
    longest = _log_int(rng, 1, min(8192, rows))
    case = {'op': op, 'type': kind, 'seqs': _log_int(rng, 1, max(1, min(512, rows // longest))), 'longest': longest,
            'ragged': rng.random() < 0.5, 'width': width, 'grad': rng.random() < 0.6}
    return {**case, 'taps': rng.randint(1, 8)} if op == 'conv' else {**case, 'states': states, 'groups': groups}


def _lengths(case):
    """The sequences' lengths: the longest everywhere, or anything from 0 up to it (one of them is the longest)."""
    if not case['ragged']:
        return [case['longest']] * case['seqs']
    rng = random.Random(case['seqs'] * 10007 + case['longest'])
    return [case['longest']] + [rng.randint(0, case['longest']) for _ in range(case['seqs'] - 1)]


def _offsets(case):
    off = [0]
    for n in _lengths(case):
        off.append(off[-1] + n)
    return off


def _randn(g, *shape):
    return torch.randn(*shape, device=g.device, generator=g)


def _weights(g, case):
    """The parameters of a scan: rates spread as usual (A from -1 to -N, steps between 1e-3 and 1e-1 through dt_bias)."""
    width, n = case['width'], case['states']
    a = -(torch.arange(1, n + 1, device=g.device).float() * (0.5 + torch.rand(width, 1, device=g.device, generator=g)))
    step = torch.exp(torch.rand(width, device=g.device, generator=g) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    return a.contiguous(), 1.0 + 0.1 * _randn(g, width), step + torch.log(-torch.expm1(-step))


def prepare(case, seed):
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(seed)
    t, op, s = TYPES[case['type']], case['op'], {'case': dict(case)}
    if op == 'norm':
        rows, width = case['rows'], case['width']
        s['x'] = (_randn(g, rows, width) * 1.5 + 0.5 * _randn(g, rows, 1)).to(t)
        s['w'], s['b'] = 1.0 + 0.2 * _randn(g, width), 0.2 * _randn(g, width)
        s['dy'] = _randn(g, rows, width).to(t) if case['grad'] else None
        leaves = ('x', 'w', 'b')
    elif op in ('conv', 'conv_step'):
        width, taps = case['width'], case['taps']
        s['w'], s['b'] = _randn(g, width, taps) / math.sqrt(taps), 0.1 * _randn(g, width)
        leaves = ('x', 'w', 'b')
        if op == 'conv_step':
            s['x'] = _randn(g, case['seqs'], width).to(t)
            s['state'] = _randn(g, case['seqs'], taps - 1, width).to(t)
            s['next'] = torch.empty_like(s['state'])
    else:
        width, n, groups = case['width'], case['states'], case['groups']
        s['A'], s['D'], s['bias'] = _weights(g, case)
        leaves = ('x', 'dt', 'A', 'B', 'C', 'D', 'z', 'bias', 'h0')
        lead = (case['seqs'],) if op == 'scan_step' else (_offsets(case)[-1],)
        s['x'], s['z'] = _randn(g, *lead, width).to(t), _randn(g, *lead, width).to(t)
        s['dt'] = _randn(g, *lead, width).to(t)
        s['B'], s['C'] = _randn(g, *lead, groups, n).to(t), _randn(g, *lead, groups, n).to(t)
        s['h0'] = 0.3 * _randn(g, case['seqs'], width, n)
        if op == 'scan_step':
            s['next'] = torch.empty_like(s['h0'])
    if op in ('conv', 'scan'):
        off = _offsets(case)
        s['off'] = torch.tensor(off, dtype=torch.int32, device=dev)
        s['longest'] = case['longest']
        s['starts'] = torch.tensor([o for o, e in zip(off, off[1:]) if e > o], device=dev)
        if op == 'conv':
            s['x'] = _randn(g, off[-1], width).to(t)
        s['dy'] = _randn(g, off[-1], width).to(t) if case['grad'] else None
        # a user with sequences of one length holds them as [sequences, length, width], any other packed with offsets
        if not case['ragged']:
            for k in ('x', 'dt', 'z', 'B', 'C', 'dy'):
                if s.get(k) is not None:
                    s[k] = s[k].reshape(case['seqs'], case['longest'], *s[k].shape[1:])
        if op == 'scan' and not case['grad']:
            s['h0'] = None
    if case.get('grad'):
        s['leaves'] = [s[k].requires_grad_() for k in leaves if k in s]
    return s


def run(state):
    op = state['case']['op']
    if own:
        return {'norm': _own_norm, 'conv': _own_conv, 'conv_step': _own_conv_step, 'scan': _own_scan, 'scan_step': _own_scan_step}[op](state)
    with torch.no_grad():
        return {'norm': _norm, 'conv': _conv, 'conv_step': _conv_step, 'scan': _scan, 'scan_step': _scan_step}[op](state)


# ------------------------------------------------------------------ the framework's calls

def _own_norm(s):
    from ps_vae_amd import ops
    y = ops.layer_norm(s['x'], s['w'], s['b'], EPS)
    return [y, *torch.autograd.grad(y, s['leaves'], s['dy'])] if s['dy'] is not None else [y]


def _own_conv(s):
    from ps_vae_amd import ops
    y = ops.causal_conv(s['x'], s['w'], s['b'], silu=True, seq_off=s['off'] if s['case']['ragged'] else None)
    return [y, *torch.autograd.grad(y, s['leaves'], s['dy'])] if s['dy'] is not None else [y]


def _own_conv_step(s):
    from ps_vae_amd import ops
    return list(ops.causal_conv_step(s['x'], s['state'], s['w'], s['b'], silu=True, state_out=s['next']))


def _own_scan(s):
    from ps_vae_amd import ops
    y, last = ops.selective_scan(s['x'], s['dt'], s['A'], s['B'], s['C'], D=s['D'], z=s['z'], dt_bias=s['bias'], softplus=True,
                                 h0=s['h0'], seq_off=s['off'] if s['case']['ragged'] else None, return_state=True)
    return [y, last, *torch.autograd.grad(y, s['leaves'], s['dy'])] if s['dy'] is not None else [y, last]


def _own_scan_step(s):
    from ps_vae_amd import ops
    return list(ops.selective_scan_step(s['x'], s['dt'], s['A'], s['B'], s['C'], s['h0'], D=s['D'], z=s['z'], dt_bias=s['bias'],
                                        softplus=True, state_out=s['next']))


# ------------------------------------------------------------------ the plain forms

def _norm(s):
    t = s['x'].dtype
    x = s['x'].float()
    xc = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    xhat = xc * rstd
    y = (xhat * s['w'] + s['b']).to(t)
    if s['dy'] is None:
        return [y]
    dy = s['dy'].float()
    g = dy * s['w']
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return [y, dx.to(t), (dy * xhat).sum(0), dy.sum(0)]


def _taps(s, x):
    """[taps, rows, width]: row t - (taps - 1) + k of the same sequence, zero in front of it."""
    taps, rows = s['case']['taps'], x.shape[0]
    pos = torch.arange(rows, device=x.device)
    off = s['off'].long()
    inside = pos - off[torch.searchsorted(off, pos, right=True) - 1]
    back = torch.arange(taps - 1, -1, -1, device=x.device)[:, None]
    return x[(pos - back).clamp(min=0)] * (inside >= back)[..., None], inside, back


def _conv(s):
    t, shape = s['x'].dtype, s['x'].shape
    x = s['x'].reshape(-1, shape[-1]).float()
    window, inside, back = _taps(s, x)
    pre = (window * s['w'].t()[:, None]).sum(0) + s['b']
    sig = torch.sigmoid(pre)
    y = (pre * sig).to(t).reshape(shape)
    if s['dy'] is None:
        return [y]
    dpre = s['dy'].reshape(-1, shape[-1]).float() * sig * (1 + pre * (1 - sig))
    # row t's value was tap k's factor in row t + back, if that row exists and belongs to the same sequence
    pos = torch.arange(x.shape[0], device=x.device)
    to = (pos + back).clamp(max=x.shape[0] - 1)
    same = (pos + back < x.shape[0]) & (inside[to] >= back)
    dx = (dpre[to] * same[..., None] * s['w'].t()[:, None]).sum(0)
    return [y, dx.to(t).reshape(shape), (window * dpre).sum(1).t(), dpre.sum(0)]


def _conv_step(s):
    t = s['x'].dtype
    window = torch.cat([s['state'], s['x'][:, None]], 1)
    pre = (window.float() * s['w'].t()).sum(1) + s['b']
    return [(pre * torch.sigmoid(pre)).to(t), window[:, 1:]]


def _doubling(a, b, longest):
    """h[t] = a[t] h[t-1] + b[t] over the rows, by doubling the stretch that every row has summed."""
    step = 1
    while step < longest:
        b = torch.cat([b[:step], torch.addcmul(b[step:], a[step:], b[:-step])])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(v.clamp(max=20))))


def _scan(s):
    t, shape, (width, n) = s['x'].dtype, s['x'].shape, s['A'].shape
    groups = s['case']['groups']
    flat = lambda v: v.reshape(-1, width).float()  # noqa: E731
    spread = lambda v: v.reshape(-1, groups, 1, n).float().expand(-1, -1, width // groups, -1).reshape(-1, width, n)  # noqa: E731
    x, z, v = flat(s['x']), flat(s['z']), flat(s['dt']) + s['bias']
    B, C = spread(s['B']), spread(s['C'])
    off, rows = s['off'].long(), x.shape[0]
    full = off[1:] > off[:-1]
    starts, ends = s['starts'], off[1:][full] - 1
    delta = _softplus(v)
    a = torch.exp(delta[..., None] * s['A'])
    b = (delta * x)[..., None] * B
    if s['h0'] is not None:
        b[starts] += a[starts] * s['h0'][full]
    cut = torch.ones(rows, 1, 1, device=x.device)
    cut[starts] = 0
    h = _doubling(a * cut, b, s['longest'])
    last = torch.zeros(off.numel() - 1, width, n, device=x.device) if s['h0'] is None else s['h0'].clone()
    last[full] = h[ends]
    y = (h * C).sum(-1) + s['D'] * x
    sig = torch.sigmoid(z)
    out = [(y * z * sig).to(t).reshape(shape), last]
    if s['dy'] is None:
        return out
    dout = flat(s['dy'])
    dy = dout * z * sig
    dz = dout * y * sig * (1 + z * (1 - sig))
    # gradient of the states: G[t] = C[t] dy[t] + a[t+1] G[t+1] inside a sequence
    ahead = torch.cat([(a * cut)[1:], torch.zeros_like(a[:1])])
    G = _doubling(ahead.flip(0), (C * dy[..., None]).flip(0), s['longest']).flip(0)
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    before[starts] = s['h0'][full]
    decayed = G * a * before
    by_b = (G * B).sum(-1)
    ddelta = by_b * x + (decayed * s['A']).sum(-1)
    dv = ddelta * torch.where(v > 20, torch.ones_like(v), torch.sigmoid(v))
    dx = by_b * delta + s['D'] * dy
    dA = (decayed * delta[..., None]).sum(0)
    gather = lambda q: q.reshape(rows, groups, width // groups, n).sum(2).to(t).reshape(s['B'].shape)  # noqa: E731
    dB, dC = gather(G * (delta * x)[..., None]), gather(h * dy[..., None])
    dh0 = torch.zeros_like(s['h0'])
    dh0[full] = (G * a)[starts]
    return out + [dx.to(t).reshape(shape), dv.to(t).reshape(shape), dA, dB, dC, (dy * x).sum(0), dz.to(t).reshape(shape), dv.sum(0), dh0]


def _scan_step(s):
    t, (width, n) = s['x'].dtype, s['A'].shape
    spread = lambda v: v.float().repeat_interleave(width // s['case']['groups'], 1)  # noqa: E731
    x, z = s['x'].float(), s['z'].float()
    delta = _softplus(s['dt'].float() + s['bias'])
    h = torch.exp(delta[..., None] * s['A']) * s['h0'] + (delta * x)[..., None] * spread(s['B'])
    y = (h * spread(s['C'])).sum(-1) + s['D'] * x
    return [(y * z * torch.sigmoid(z)).to(t), h]


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    e, op = BYTES[case['type']], case['op']
    if op == 'norm':
        cells = case['rows'] * case['width']
        return {'bytes': cells * e * (4 if case['grad'] else 2) + case['width'] * 4 * (4 if case['grad'] else 2),
                'flops': cells * (18 if case['grad'] else 7)}
    if op == 'conv_step':
        cells = case['seqs'] * case['width']
        return {'bytes': cells * e * 2 * case['taps'] + case['width'] * 4 * (case['taps'] + 1), 'flops': cells * (2 * case['taps'] + 4)}
    if op == 'conv':
        cells = sum(_lengths(case)) * case['width']
        return {'bytes': cells * e * (4 if case['grad'] else 2) + case['width'] * 4 * (case['taps'] + 1) * (2 if case['grad'] else 1),
                'flops': cells * (case['taps'] * (8 if case['grad'] else 2) + 8)}
    width, n, groups = case['width'], case['states'], case['groups']
    states, weights = case['seqs'] * width * n * 4, width * (n + 2) * 4
    if op == 'scan_step':
        return {'bytes': case['seqs'] * (width * 4 + 2 * groups * n) * e + 2 * states + weights, 'flops': case['seqs'] * width * (n * 7 + 10)}
    rows = sum(_lengths(case))
    if case['grad']:  # x, dt, z, dy and B, C in; y, dx, ddt, dz and dB, dC out; h0, its gradient and the last state
        return {'bytes': rows * (8 * width + 4 * groups * n) * e + 3 * states + 2 * weights, 'flops': rows * width * (n * 27 + 40)}
    return {'bytes': rows * (4 * width + 2 * groups * n) * e + states + weights, 'flops': rows * width * (n * 7 + 10)}


# ------------------------------------------------------------------ the definitions in 64 bits

def _padded(case, rows):
    """[sequences, longest, ...] with every sequence's rows in front."""
    out = torch.zeros(case['seqs'], case['longest'], *rows.shape[1:], dtype=torch.float64, device=rows.device)
    off = _offsets(case)
    for i, (o, e) in enumerate(zip(off, off[1:])):
        out[i, :e - o] = rows[o:e]
    return out


def _packed(case, padded):
    return torch.cat([padded[i, :n] for i, n in enumerate(_lengths(case))])


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    op = case['op']
    if op == 'norm':
        keys = ('x', 'w', 'b')
        leaf = [d[k].requires_grad_() for k in keys]
        x = leaf[0]
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + EPS) * leaf[1] + leaf[2]
        out = [y.detach()]
        return out + list(torch.autograd.grad(y, leaf, d['dy'])) if case['grad'] else out
    if op == 'conv_step':
        pre = d['b'] + d['w'][:, -1] * d['x']
        for k in range(case['taps'] - 1):
            pre = pre + d['w'][:, k] * d['state'][:, k]
        return [pre / (1 + torch.exp(-pre)), torch.cat([d['state'], d['x'][:, None]], 1)[:, 1:]]
    if op == 'conv':
        shape, taps = d['x'].shape, case['taps']
        x = _padded(case, d['x'].reshape(-1, case['width'])).requires_grad_()
        leaf = [x, d['w'].requires_grad_(), d['b'].requires_grad_()]
        pre = leaf[2].expand_as(x)
        for k in range(taps):
            back = taps - 1 - k
            if back < case['longest']:
                pre = pre + torch.nn.functional.pad(x[:, :case['longest'] - back], (0, 0, back, 0)) * leaf[1][:, k]
        y = pre / (1 + torch.exp(-pre))
        out = [_packed(case, y.detach()).reshape(shape)]
        if not case['grad']:
            return out
        dx, dw, db = torch.autograd.grad(y, leaf, _padded(case, d['dy'].reshape(-1, case['width'])))
        return out + [_packed(case, dx).reshape(shape), dw, db]
    width, n, groups = case['width'], case['states'], case['groups']
    softplus = lambda v: torch.logaddexp(v, torch.zeros_like(v))  # noqa: E731
    spread = lambda v: v.repeat_interleave(width // groups, -2)  # noqa: E731
    if op == 'scan_step':
        delta = softplus(d['dt'] + d['bias']).unsqueeze(-1)
        h = torch.exp(delta * d['A']) * d['h0'] + delta * d['x'].unsqueeze(-1) * spread(d['B'])
        y = torch.einsum('sdn,sdn->sd', h, spread(d['C'])) + d['D'] * d['x']
        return [y * d['z'] / (1 + torch.exp(-d['z'])), h]
    if case['longest'] * case['seqs'] * width * n * 8 > 24e9:
        return None
    return _exact_scan(case, d, softplus, spread)


def _exact_scan(case, d, softplus, spread):
    width, n, groups = case['width'], case['states'], case['groups']
    shape = d['x'].shape
    x, z, dt = (_padded(case, d[k].reshape(-1, width)) for k in ('x', 'z', 'dt'))
    B, C = (_padded(case, d[k].reshape(-1, groups, n)) for k in ('B', 'C'))
    long = torch.tensor(_lengths(case), device=x.device)
    v = dt + d['bias']
    delta = softplus(v)
    h = d['h0'] if 'h0' in d else torch.zeros(case['seqs'], width, n, dtype=torch.float64, device=x.device)
    first, steps, y = h, case['longest'], torch.empty_like(x)
    kept = torch.empty(steps, *h.shape, dtype=h.dtype, device=h.device) if case['grad'] else None
    for i in range(steps):
        moved = torch.exp(delta[:, i, :, None] * d['A']) * h + (delta[:, i] * x[:, i])[..., None] * spread(B[:, i])
        h = torch.where((i < long)[:, None, None], moved, h)
        if kept is not None:
            kept[i] = h
        y[:, i] = (h * spread(C[:, i])).sum(-1) + d['D'] * x[:, i]
    gate = z / (1 + torch.exp(-z))
    pack = lambda q: _packed(case, q)  # noqa: E731
    out = [pack(y * gate).reshape(shape), h]
    if not case['grad']:
        return out
    dout = _padded(case, d['dy'].reshape(-1, width))
    sig = 1 / (1 + torch.exp(-z))
    dy, dz = dout * gate, dout * y * (sig + gate * (1 - sig))
    dx, ddelta, dB, dC = torch.empty_like(x), torch.empty_like(x), torch.empty_like(B), torch.empty_like(C)
    dA, carry = torch.zeros_like(d['A']), torch.zeros_like(h)
    split = lambda q: q.reshape(q.shape[0], groups, width // groups, n).sum(2)  # noqa: E731
    for i in reversed(range(steps)):
        live = (i < long)[:, None, None]
        G = (carry + spread(C[:, i]) * dy[:, i, :, None]) * live
        a = torch.exp(delta[:, i, :, None] * d['A'])
        dC[:, i], dB[:, i] = split(kept[i] * dy[:, i, :, None]), split(G * (delta[:, i] * x[:, i])[..., None])
        inflow = (G * spread(B[:, i])).sum(-1)
        decay = G * a * (kept[i - 1] if i else first)
        dx[:, i] = inflow * delta[:, i] + d['D'] * dy[:, i]
        ddelta[:, i] = inflow * x[:, i] + (decay * d['A']).sum(-1)
        dA += (decay * delta[:, i, :, None]).sum(0)
        carry = torch.where(live, a * G, carry)
    dv = ddelta / (1 + torch.exp(-v))
    back = lambda q, like: pack(q).reshape(like.shape)  # noqa: E731
    alive = (torch.arange(steps, device=x.device) < long[:, None])[..., None]
    return out + [back(dx, d['x']), back(dv, d['x']), dA, back(dB, d['B']), back(dC, d['C']), (dy * x * alive).sum((0, 1)),
                  back(dz, d['x']), (dv * alive).sum((0, 1)), carry * (long > 0)[:, None, None]]
