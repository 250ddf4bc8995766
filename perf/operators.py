"""Cases and plain forms of the operators that train and serve a head over sparse rows: row
normalisation with its gradients, counter-based dropout with its gradient, and the gated
linear recurrence over serialised rows (forward, backward, one step).

Run as plain torch operations (``own`` false) or through this package's operators (``own``
true). A row is one voxel of a ``SparseTensor``; sequences are the clouds of a batch.
"""

from __future__ import annotations

import math

import torch

own = False

_TYPES = {'fp16': torch.float16, 'fp32': torch.float32}
_SIZE = {'fp16': 2, 'fp32': 4}


def listed():
    return [
        # globally pooled features of eight clouds in a training step: latency
        {'name': 'layer_norm pooled', 'op': 'norm', 'kind': 'layer', 'dtype': 'fp32', 'rows': 8, 'channels': 256},
        # every voxel of an 8 x 120,000 voxel batch at the 64-channel level
        {'name': 'layer_norm clouds', 'op': 'norm', 'kind': 'layer', 'dtype': 'fp16', 'rows': 960000, 'channels': 64},
        # an odd number of rows at the width of the 96 -> 192 block
        {'name': 'rms_norm block', 'op': 'norm', 'kind': 'rms', 'dtype': 'fp16', 'rows': 240001, 'channels': 192},
        # few, wide rows in float32
        {'name': 'layer_norm wide', 'op': 'norm', 'kind': 'layer', 'dtype': 'fp32', 'rows': 30011, 'channels': 1000},
        # 20-channel logits of a small cloud: odd, unaligned, latency
        {'name': 'dropout logits', 'op': 'dropout', 'dtype': 'fp32', 'rows': 2003, 'channels': 20, 'p': 0.5,
         'residual': False},
        # the residual branch of a block over the whole batch
        {'name': 'dropout residual clouds', 'op': 'dropout', 'dtype': 'fp16', 'rows': 960000, 'channels': 64,
         'p': 0.1, 'residual': True},
        # float32 features without a residual
        {'name': 'dropout fp32', 'op': 'dropout', 'dtype': 'fp32', 'rows': 240000, 'channels': 96, 'p': 0.25,
         'residual': False},
        # one training pass over eight whole clouds
        {'name': 'recurrence train clouds', 'op': 'recurrence', 'dtype': 'fp16', 'rows': 960000, 'channels': 64,
         'sequences': 8, 'padding': 0, 'train': True, 'reverse': False},
        # serving one cloud as one long sequence, last row first
        {'name': 'recurrence serve cloud', 'op': 'recurrence', 'dtype': 'fp16', 'rows': 120000, 'channels': 128,
         'sequences': 1, 'padding': 0, 'train': False, 'reverse': True},
        # many short ragged windows in a buffer with unused rows behind the last one
        {'name': 'recurrence train windows', 'op': 'recurrence', 'dtype': 'fp32', 'rows': 200000, 'channels': 96,
         'sequences': 5003, 'padding': 777, 'train': True, 'reverse': True},
        # one new row for each of eight streams: latency
        {'name': 'recurrence step', 'op': 'step', 'dtype': 'fp16', 'rows': 8, 'channels': 256},
        # one new row for each of many streams
        {'name': 'recurrence step many', 'op': 'step', 'dtype': 'fp32', 'rows': 16411, 'channels': 192},
    ]


_LARGEST = 960000 * 64


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(('norm', 'norm', 'dropout', 'recurrence', 'recurrence', 'step'))
    dtype = rng.choice(('fp16', 'fp32'))
    # normalising a row of a handful of channels leaves its gradient to cancellation
    channels = rng.choice((_log(rng, 8 if op == 'norm' else 1, 1024), 8 * _log(rng, 1, 128)))
    rows = _log(rng, 1, min(960000, _LARGEST * 2 // (channels * _SIZE[dtype])))
    case = {'op': op, 'dtype': dtype, 'rows': rows, 'channels': channels}
    if op == 'norm':
        case['kind'] = rng.choice(('layer', 'rms'))
    elif op == 'dropout':
        case['p'] = round(rng.uniform(0.05, 0.9), 3)
        case['residual'] = rng.random() < 0.5
    elif op == 'recurrence':
        case['padding'] = rng.choice((0, rng.randrange(0, rows // 4 + 1)))
        case['sequences'] = _log(rng, 1, max(1, rows // 3))
        case['train'] = rng.random() < 0.6
        case['reverse'] = rng.random() < 0.5
    return case


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #


def prepare(case, seed):
    device = torch.device('cuda')
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = _TYPES[case['dtype']]
    rows, channels = case['rows'], case['channels']

    def normal(*shape, scale=1.0, shift=0.0, to=dtype):
        return (torch.randn(shape, generator=gen, device=device) * scale + shift).to(to)

    state = {'case': case}
    # features after a few layers: channels with their own offset and width
    width = torch.rand(channels, generator=gen, device=device) + 0.5
    shift = torch.randn(channels, generator=gen, device=device)
    state['feats'] = (normal(rows, channels, to=torch.float32) * width + shift).to(dtype)
    if case['op'] == 'norm':
        state['weight'] = normal(channels, scale=0.2, shift=1.0)
        state['bias'] = normal(channels, scale=0.2) if case['kind'] == 'layer' else None
        state['grad'] = normal(rows, channels)
    elif case['op'] == 'dropout':
        state['residual'] = normal(rows, channels) if case['residual'] else None
        state['grad'] = normal(rows, channels)
        state['seed'] = (seed * 0x9E3779B97F4A7C15 + 12345) % (1 << 63)
        state['offset'] = 3
    else:
        # forget-gate logits: the bias spreads the channels' memory from a few rows to hundreds
        spread = torch.linspace(0.0, 5.0, channels, device=device)
        state['gate'] = (normal(rows, channels, to=torch.float32) + spread).to(dtype)
        sequences = rows if case['op'] == 'step' else case['sequences']
        state['initial'] = normal(sequences, channels, scale=0.5, to=torch.float32)
        if case['op'] == 'recurrence':
            used = rows - case['padding']
            cuts = torch.randint(0, used + 1, (sequences - 1,), generator=gen, device=device).sort().values
            ends = torch.tensor([0, used], device=device)
            state['offsets'] = torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32)
            state['grad'] = normal(rows, channels)
            state['grad_final'] = normal(sequences, channels, to=torch.float32)
    if own:
        from mlx_lattice_b200.core import SparseTensor

        coords = torch.zeros((rows, 4), dtype=torch.int32, device=device)
        coords[:, 1] = torch.arange(rows, dtype=torch.int32, device=device)
        if case['op'] in ('norm', 'dropout') or case.get('train'):
            for name in ('feats', 'weight', 'bias', 'gate', 'initial'):
                if state.get(name) is not None:
                    state[name].requires_grad_(True)
        state['x'] = SparseTensor(coords, state['feats'])
    return state


def work(case):
    size, n, c = _SIZE[case['dtype']], case['rows'], case['channels']
    if case['op'] == 'norm':
        vectors = 4 if case['kind'] == 'layer' else 2
        # x, dy in; y, dx out
        return {'bytes': 4 * n * c * size + vectors * c * size, 'flops': 18 * n * c}
    if case['op'] == 'dropout':
        # x, dy (and the residual) in; y, dx out
        return {'bytes': (5 if case['residual'] else 4) * n * c * size, 'flops': 4 * n * c}
    if case['op'] == 'step':
        return {'bytes': 3 * n * c * size + 8 * n * c, 'flops': 8 * n * c}
    states = case['sequences'] * c * 4
    if case['train']:
        # x, gate, dy in; h, dx, dgate out; initial and final state with their gradients
        return {'bytes': 6 * n * c * size + 4 * states, 'flops': 25 * n * c}
    return {'bytes': 3 * n * c * size + 2 * states, 'flops': 8 * n * c}


# --------------------------------------------------------------------------- #
# one pass
# --------------------------------------------------------------------------- #


def run(state):
    op = state['case']['op']
    if own:
        return {'norm': _own_norm, 'dropout': _own_dropout, 'recurrence': _own_recurrence, 'step': _own_step}[op](state)
    return {'norm': _norm, 'dropout': _dropout, 'recurrence': _recurrence, 'step': _step}[op](state)


def _own_norm(s):
    from mlx_lattice_b200 import ops

    if s['case']['kind'] == 'rms':
        y = ops.rms_norm(s['x'], weight=s['weight']).feats
        dx, dw = torch.autograd.grad(y, (s['feats'], s['weight']), s['grad'])
        return {'y': y, 'dx': dx, 'dw': dw}
    y = ops.layer_norm(s['x'], weight=s['weight'], bias=s['bias']).feats
    dx, dw, db = torch.autograd.grad(y, (s['feats'], s['weight'], s['bias']), s['grad'])
    return {'y': y, 'dx': dx, 'dw': dw, 'db': db}


def _own_dropout(s):
    from mlx_lattice_b200 import ops

    y = ops.dropout(s['x'], p=s['case']['p'], training=True, seed=s['seed'], offset=s['offset'],
                    residual=s['residual']).feats
    dx, = torch.autograd.grad(y, (s['feats'],), s['grad'])
    return {'y': y, 'dx': dx}


def _own_recurrence(s):
    from mlx_lattice_b200 import ops

    y, final = ops.gated_recurrence(s['x'], s['gate'], initial_state=s['initial'], offsets=s['offsets'],
                                    reverse=s['case']['reverse'], return_state=True)
    if not s['case']['train']:
        return {'h': y.feats, 'final': final}
    dx, dgate, dinitial = torch.autograd.grad(
        (y.feats, final), (s['feats'], s['gate'], s['initial']), (s['grad'], s['grad_final']))
    return {'h': y.feats, 'final': final, 'dx': dx, 'dgate': dgate, 'dinitial': dinitial}


def _own_step(s):
    from mlx_lattice_b200 import ops

    y, state = ops.gated_recurrence_step(s['x'], s['gate'], s['initial'])
    return {'h': y.feats, 'state': state}


# ---- plain forms ------------------------------------------------------------- #


def _norm(s):
    x, dy, w = s['feats'].float(), s['grad'].float(), s['weight'].float()
    dtype = s['feats'].dtype
    if s['case']['kind'] == 'layer':
        x = x - x.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-5)
    xhat = x * r
    g = dy * w
    dx = g - xhat * (g * xhat).mean(1, keepdim=True)
    out = {'dw': (dy * xhat).sum(0, dtype=torch.float64).to(dtype)}
    if s['case']['kind'] == 'layer':
        dx = dx - g.mean(1, keepdim=True)
        out['db'] = dy.sum(0, dtype=torch.float64).to(dtype)
        out['y'] = (xhat * w + s['bias'].float()).to(dtype)
    else:
        out['y'] = (xhat * w).to(dtype)
    out['dx'] = (dx * r).to(dtype)
    return out


_LOW = 0xFFFFFFFF


def _philox(index, offset, seed):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2,
    3", 2011): the four 32-bit words of each 64-bit counter ``index``, as int64 tensors. The
    products wrap modulo 2^64, which keeps both 32-bit halves right."""
    c0, c1 = index & _LOW, index >> 32
    c2 = torch.full_like(index, offset & _LOW)
    c3 = torch.full_like(index, (offset >> 32) & _LOW)
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & _LOW) ^ c1 ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ c3 ^ k1, a & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return c0, c1, c2, c3


def _dropout(s):
    x, dtype, p = s['feats'], s['feats'].dtype, s['case']['p']
    total = x.numel()
    index = torch.arange((total + 3) // 4, dtype=torch.int64, device=x.device)
    words = torch.stack(_philox(index, s['offset'], s['seed']), dim=1).reshape(-1)[:total].view(x.shape)
    keep = words >= int(math.floor(p * 4294967296.0 + 0.5))
    scale = 1.0 / (1.0 - p)
    y = torch.where(keep, x.float() * scale, 0.0)
    if s['residual'] is not None:
        y = y + s['residual'].float()
    return {'y': y.to(dtype), 'dx': torch.where(keep, s['grad'].float() * scale, 0.0).to(dtype)}


def _doubling(a, b):
    """h[t] = a[t] h[t - 1] + b[t] with h[-1] = 0 for all rows at once, by doubling."""
    step, n = 1, a.shape[0]
    while step < n:
        b = torch.cat([b[:step], torch.addcmul(b[step:], a[step:], b[:-step])])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _recurrence(s):
    case, dtype = s['case'], s['feats'].dtype
    x, z, off, initial = s['feats'].float(), s['gate'].float(), s['offsets'].long(), s['initial']
    n = x.shape[0]
    dy, dfinal = s['grad'].float(), s['grad_final']
    if case['reverse']:
        x, z, dy = x.flip(0), z.flip(0), dy.flip(0)
        off, initial, dfinal = n - off.flip(0), initial.flip(0), dfinal.flip(0)
    rows = torch.arange(n, device=x.device)
    begin, end, full = off[:-1], off[1:], (off[1:] > off[:-1])[:, None]
    seq = torch.searchsorted(end, rows, right=True).clamp(max=end.numel() - 1)
    live = ((rows >= off[0]) & (rows < off[-1]))[:, None]
    head = ((rows == begin[seq])[:, None]) & live
    tail = ((rows == end[seq] - 1)[:, None]) & live
    a, keep = torch.sigmoid(z), torch.sigmoid(-z)
    b = keep * x
    h = _doubling(torch.where(head | ~live, 0.0, a), torch.where(live, torch.where(head, b + a * initial[seq], b), 0.0))
    final = torch.where(full, h[(end - 1).clamp(min=0)], initial)
    out = {'h': h, 'final': final}
    if case['train']:
        before = torch.where(head, initial[seq], torch.roll(h, 1, 0))
        dh = torch.where(live, dy, 0.0) + torch.where(tail, dfinal[seq], 0.0)
        carry = torch.where(tail | ~live, 0.0, torch.roll(a, -1, 0))
        dh = _doubling(carry.flip(0), dh.flip(0)).flip(0)
        out['dx'] = torch.where(live, keep * dh, 0.0)
        out['dgate'] = torch.where(live, a * keep * dh * (before - x), 0.0)
        out['dinitial'] = torch.where(full, (a * dh)[begin.clamp(max=n - 1)], dfinal)
    if case['reverse']:
        out = {k: v.flip(0) for k, v in out.items()}
    return {k: v if k in ('final', 'dinitial') else v.to(dtype) for k, v in out.items()}


def _step(s):
    a = torch.sigmoid(s['gate'].float())
    h = a * s['initial'] + (1.0 - a) * s['feats'].float()
    return {'h': h.to(s['feats'].dtype), 'state': h}


# ---- in 64 bits -------------------------------------------------------------- #


def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    return {'norm': _exact_norm, 'dropout': _exact_dropout, 'recurrence': _exact_recurrence,
            'step': _exact_step}[case['op']](s)


def _exact_norm(s):
    """The gradient as the transposed Jacobian of (x - m) / sqrt(v + eps), term by term."""
    x, w, dy = s['feats'].double(), s['weight'].double(), s['grad'].double()
    c = x.shape[1]
    layer = s['case']['kind'] == 'layer'
    m = x.sum(1, keepdim=True) / c if layer else torch.zeros_like(x[:, :1])
    v = (x - m).pow(2).sum(1, keepdim=True) / c
    sd = (v + 1e-5).sqrt()
    up = dy * w
    dv = -0.5 * (up * (x - m)).sum(1, keepdim=True) / (sd * (v + 1e-5))
    dx = up / sd + dv * 2.0 * (x - m) / c
    if not layer:
        return {'y': x / sd * w, 'dx': dx, 'dw': (dy * x / sd).sum(0)}
    dm = -(up / sd).sum(1, keepdim=True) - dv * 2.0 * (x - m).sum(1, keepdim=True) / c
    return {'y': (x - m) / sd * w + s['bias'].double(), 'dx': dx + dm / c,
            'dw': (dy * (x - m) / sd).sum(0), 'db': dy.sum(0)}


def _times(word, constant):
    """(high, low) 32 bits of a 32 x 32 bit product, from 16-bit limbs."""
    x0, x1, y0, y1 = word % 65536, word // 65536, constant % 65536, constant // 65536
    low = x0 * y0
    middle = x1 * y0 + low // 65536
    middle2 = x0 * y1 + middle % 65536
    return x1 * y1 + middle // 65536 + middle2 // 65536, (middle2 % 65536) * 65536 + low % 65536


def _exact_dropout(s):
    x, p = s['feats'].double(), s['case']['p']
    shape, total = x.shape, x.numel()
    at = torch.arange(-(-total // 4), device=x.device)
    ctr = [at % 2 ** 32, at // 2 ** 32, at * 0 + s['offset'] % 2 ** 32, at * 0 + s['offset'] // 2 ** 32]
    for turn in range(10):
        key = ((s['seed'] + turn * 0x9E3779B9) % 2 ** 32, (s['seed'] // 2 ** 32 + turn * 0xBB67AE85) % 2 ** 32)
        h0, l0 = _times(ctr[0], 0xD2511F53)
        h1, l1 = _times(ctr[2], 0xCD9E8D57)
        ctr = [h1 ^ ctr[1] ^ key[0], l1, h0 ^ ctr[3] ^ key[1], l0]
    dropped = (torch.stack(ctr, 1).flatten()[:total] < round(p * 2 ** 32)).view(shape)
    y = (x / (1.0 - p)).masked_fill(dropped, 0.0)
    dx = (s['grad'].double() / (1.0 - p)).masked_fill(dropped, 0.0)
    return {'y': y if s['residual'] is None else y + s['residual'].double(), 'dx': dx}


def _walk(a, b):
    """h[t] = a[t] h[t - 1] + b[t] with h[-1] = 0, one row after the other within blocks of
    rows, then one block after the other."""
    n, c = a.shape
    block = max(1, int(math.sqrt(n)))
    count = -(-n // block)
    pad = count * block - n
    a = torch.cat([a, a.new_ones(pad, c)]).view(count, block, c)
    b = torch.cat([b, b.new_zeros(pad, c)]).view(count, block, c)
    h, p = torch.empty_like(b), torch.empty_like(a)
    h[:, 0], p[:, 0] = b[:, 0], a[:, 0]
    for t in range(1, block):
        h[:, t] = a[:, t] * h[:, t - 1] + b[:, t]
        p[:, t] = a[:, t] * p[:, t - 1]
    state = torch.zeros_like(h[0, 0])
    before = torch.empty_like(h[:, 0])
    for k in range(count):
        before[k] = state
        state = p[k, -1] * state + h[k, -1]
    h += p * before[:, None]
    return h.view(-1, c)[:n]


def _exact_recurrence(s):
    case = s['case']
    x, z, initial = s['feats'].double(), s['gate'].double(), s['initial'].double()
    n, c = x.shape
    back = case['reverse']
    # sequences as (first row, last row) in the order of time, those without rows apart
    off = s['offsets'].long()
    lengths = off[1:] - off[:-1]
    some = torch.nonzero(lengths > 0).flatten()
    low, high = off[:-1][some], off[1:][some] - 1
    first, last = (high, low) if back else (low, high)
    used = torch.zeros(n, dtype=torch.bool, device=x.device)
    used[int(off[0]):int(off[-1])] = True
    gone = ~used[:, None]
    a = 1.0 / (1.0 + torch.exp(-z))
    rest = 1.0 / (1.0 + torch.exp(z))
    u = (rest * x).masked_fill(gone, 0.0)
    u[first] += a[first] * initial[some]
    decay = a.masked_fill(gone, 0.0)
    decay[first] = 0.0
    turn = (lambda v: v.flip(0)) if back else (lambda v: v)
    h = turn(_walk(turn(decay), turn(u)))
    final = initial.clone()
    final[some] = h[last]
    out = {'h': h, 'final': final}
    if case['train']:
        prior = torch.zeros_like(h)
        if back:
            prior[:-1] = h[1:]
        else:
            prior[1:] = h[:-1]
        prior[first] = initial[some]
        dfinal = s['grad_final'].double()
        up = s['grad'].double().masked_fill(gone, 0.0)
        up[last] += dfinal[some]
        follow = torch.zeros_like(a)
        if back:
            follow[1:] = a[:-1]
        else:
            follow[:-1] = a[1:]
        follow[last] = 0.0
        follow = follow.masked_fill(gone, 0.0)
        unturn = (lambda v: v) if back else (lambda v: v.flip(0))
        dh = unturn(_walk(unturn(follow), unturn(up)))
        out['dx'] = dh * rest
        out['dgate'] = dh * (prior - x) * a * rest
        dinitial = dfinal.clone()
        dinitial[some] = (a * dh)[first]
        out['dinitial'] = dinitial
        for name in ('dx', 'dgate'):
            out[name] = out[name].masked_fill(gone, 0.0)
    return out


def _exact_step(s):
    forget = 1.0 / (1.0 + torch.exp(-s['gate'].double()))
    h = s['feats'].double() + forget * (s['initial'].double() - s['feats'].double())
    return {'h': h, 'state': h}
