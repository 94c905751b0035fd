"""Timed cases of the state-space sequence operators: the short causal convolution, the selective scan, their single-frame forms,
layer norm and dropout (``pb_sed_amd.ops``: ``causal_conv_*``, ``selective_scan_*``, ``layer_norm_*``, ``dropout``).

``run`` computes a case in its plain form (elementary torch operations in 32 bits, rounded once at the end), or - ``own`` true -
with the calls a program makes of the framework.  Everything is time-major [T, B, channels], like the recurrent layers' buffers.
"""
import math

import torch

own = False
DEV = 'cuda'
DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def listed():
    return [
        # the layers of one training step: 32 clips of 10 s (500 frames of 20 ms) with ragged lengths, 512 inner channels
        dict(name='conv_train_f32', op='conv', train=True, dtype='f32', t=500, b=32, d=512, k=4, reverse=False, ragged=True, state=False),
        dict(name='scan_train_f32', op='scan', train=True, dtype='f32', t=500, b=32, d=512, n=16, reverse=False, ragged=True, state=False),
        # the time-reversed network on 20 s clips, half-precision activations, an odd number of frames
        dict(name='scan_train_bf16_reverse', op='scan', train=True, dtype='bf16', t=1001, b=8, d=768, n=16, reverse=True, ragged=True, state=False),
        # a recording of more than ten minutes, processed piece after piece with carried states
        dict(name='conv_prompt_bf16', op='conv', train=False, dtype='bf16', t=40000, b=2, d=1024, k=4, reverse=False, ragged=False, state=True),
        dict(name='scan_prompt_bf16_long', op='scan', train=False, dtype='bf16', t=40000, b=1, d=512, n=16, reverse=False, ragged=False, state=True),
        # a few short clips of a small detector; widths that no vector length divides
        dict(name='scan_prompt_f16_odd', op='scan', train=False, dtype='f16', t=313, b=5, d=203, n=8, reverse=False, ragged=True, state=False),
        # one frame of one live stream (latency), one frame of many
        dict(name='step_one_f32', op='step', train=False, dtype='f32', b=1, d=512, n=16, k=4),
        dict(name='step_many_bf16', op='step', train=False, dtype='bf16', b=384, d=1024, n=16, k=4),
        # the norm in front of a layer in a training step; an odd width with half-precision rows
        dict(name='norm_train_f32', op='norm', train=True, dtype='f32', rows=16000, c=256),
        dict(name='norm_train_bf16_odd', op='norm', train=True, dtype='bf16', rows=20011, c=1023),
        # dropout in front of the residual sum of a training step (forward and backward); a wide one without a residual
        dict(name='dropout_train_f32', op='dropout', train=True, dtype='f32', rows=16000, c=256, p=0.1, residual=True),
        dict(name='dropout_train_bf16', op='dropout', train=True, dtype='bf16', rows=65536, c=1000, p=0.25, residual=False),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(['conv', 'scan', 'scan', 'step', 'norm', 'dropout'])
    dtype = rng.choice(list(DTYPES))
    train = rng.random() < .6
    if op == 'step':
        return dict(op=op, train=False, dtype=dtype, b=log(1, 384), d=log(64, 1024), n=rng.choice([4, 8, 12, 16]), k=rng.choice([2, 3, 4]))
    if op in ('norm', 'dropout'):
        rows, c = log(1, 40000), log(8, 1500)
        case = dict(op=op, train=True, dtype=dtype, rows=rows, c=c)
        return dict(case, p=rng.choice([.05, .1, .25, .5]), residual=rng.random() < .5) if op == 'dropout' else case
    t, d = log(1, 2000) if train else log(1, 40000), log(64, 1024)
    b = log(1, max(1, min(48, (8_000_000 if train else 20_000_000) // (t * d))))
    case = dict(op=op, train=train, dtype=dtype, t=t, b=b, d=d, reverse=rng.random() < .3, ragged=rng.random() < .5,
                state=not train and rng.random() < .5)
    return dict(case, k=rng.choice([2, 3, 4])) if op == 'conv' else dict(case, n=rng.choice([4, 8, 12, 16]))


def lengths(case):
    """Valid frames per clip: T for all, or falling from T to about T / 2."""
    t, b = case['t'], case['b']
    return [t - (t // 2) * i // max(b - 1, 1) if case['ragged'] else t for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[case['dtype']]

    def normal(*shape, scale=1., dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    def uniform(*shape, lo, hi):
        return torch.rand(*shape, generator=g, device=DEV) * (hi - lo) + lo
    s = dict(case=case)
    if case['op'] in ('norm', 'dropout'):
        rows, c = case['rows'], case['c']
        s.update(x=normal(rows, c), dy=normal(rows, c))
        if case['op'] == 'norm':
            s['x'] = (s['x'].float() * uniform(rows, 1, lo=.2, hi=3.) + uniform(rows, 1, lo=-1., hi=1.)).to(dt)
            s.update(weight=uniform(c, lo=.5, hi=1.5), bias=normal(c, scale=.2, dtype=torch.float32), grads=torch.empty(2, c, device=DEV))
        else:
            s['rng'] = torch.tensor([(int(seed) * 0x9E3779B97F4A7C15 + 12345) % (1 << 63), 7 + int(seed) % 1000], device=DEV)
            s['residual'] = normal(rows, c) if case['residual'] else None
        return s
    b, d = case['b'], case['d']
    t = case.get('t')
    lead = (b,) if case['op'] == 'step' else (t, b)
    if case['op'] != 'step':
        s['seq_len'] = torch.tensor(lengths(case), dtype=torch.int32, device=DEV) if case['ragged'] else None
    if 'k' in case:
        k = case['k']
        s['xz'] = normal(*lead, 2 * d)                            # the input projection's output: convolution input | gate
        s['x'] = s['xz'][..., :d]
        s['weight'], s['bias'] = (uniform(d, k, lo=-1., hi=1.) / k ** .5).contiguous(), uniform(d, lo=-.5, hi=.5)
        s['conv_state'] = normal(b, k - 1, d) if case['op'] == 'step' or case['state'] else None
        if case['train']:
            s['grads'] = torch.empty(d * (k + 1), device=DEV)
    if 'n' in case:
        n = case['n']
        if case['op'] != 'step':
            s['xz'] = normal(*lead, 2 * d)
        s['z'] = s['xz'][..., d:]
        s['u'] = torch.nn.functional.silu(normal(*lead, d, dtype=torch.float32)).to(dt)
        s['delta'] = normal(*lead, d, scale=.5)
        bc = normal(*lead, 2 * n)
        s['b'], s['c'] = bc[..., :n], bc[..., n:]
        step0 = torch.exp(uniform(d, lo=math.log(1e-3), hi=math.log(1e-1)))
        s['delta_bias'] = step0 + torch.log(-torch.expm1(-step0))           # softplus(delta_bias) = step0
        s['a_log'] = (torch.log(torch.arange(1, n + 1, device=DEV, dtype=torch.float32))[None] + uniform(d, n, lo=-.2, hi=.2)).contiguous()
        s['d'] = uniform(d, lo=.5, hi=1.5)
        s['ssm_state'] = normal(b, d, n, scale=.3, dtype=torch.float32) if case['op'] == 'step' or case['state'] else None
        if case['train']:
            s['grads'] = torch.empty(d * (n + 2), device=DEV)
    if case['op'] == 'step':
        s['next_conv_state'], s['next_ssm_state'] = torch.empty_like(s['conv_state']), torch.empty_like(s['ssm_state'])
    elif case['train']:
        s['dy'] = normal(t, b, d)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _order(s, t, b):
    """(frame of scan position [T,B], clip index [1,B], valid [T,B,1])"""
    pos = torch.arange(t, device=DEV)[:, None].expand(t, b)
    lens = s['seq_len'].long()[None] if s['seq_len'] is not None else torch.full((1, b), t, device=DEV)
    valid = pos < lens
    frame = torch.where(valid, lens - 1 - pos, pos) if s['case']['reverse'] else pos
    return frame, torch.arange(b, device=DEV)[None], valid[..., None]


def _recurrence(a, x):
    """h[t] = a[t] h[t-1] + x[t] by doubling (h[-1] = 0)."""
    step = 1
    while step < len(a):
        x = torch.cat([x[:step], x[step:] + a[step:] * x[:-step]])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return x


def _plain_conv(s):
    case, w, dt = s['case'], s['weight'], s['x'].dtype
    t, b, d = s['x'].shape
    k = w.shape[1]
    frame, clip, valid = _order(s, t, b)
    x = torch.where(valid, s['x'].float()[frame, clip], 0.)
    past = s['conv_state'].float().transpose(0, 1) if case['state'] else x.new_zeros(k - 1, b, d)
    long = torch.cat([past, x])                                             # scan position p at index p + k - 1
    windows = long.unfold(0, k, 1)                                          # [T, B, D, K]
    pre = (windows * w).sum(-1) + s['bias']
    sg = torch.sigmoid(pre)
    y = torch.where(valid, pre * sg, 0.)[frame, clip].to(dt)
    if not case['train']:
        lens = s['seq_len'].long() if s['seq_len'] is not None else torch.full((b,), t, device=DEV)
        rows = lens[None] + torch.arange(k - 1, device=DEV)[:, None]
        return y, long[rows, clip].transpose(0, 1).to(dt)
    dpre = torch.where(valid, s['dy'].float()[frame, clip] * sg * (1 + pre * (1 - sg)), 0.)
    ahead = torch.cat([dpre, dpre.new_zeros(k - 1, b, d)]).unfold(0, k, 1)  # dpre[p + j], j < K: x[p] met tap K - 1 - j there
    dx = torch.where(valid, (ahead * w.flip(1)).sum(-1), 0.)[frame, clip].to(dt)
    return y, dx, (windows * dpre[..., None]).sum((0, 1)), dpre.sum((0, 1))


def _softplus(x):
    return torch.clamp(x, min=0.) + torch.log1p(torch.exp(-x.abs()))


def _plain_scan(s):
    case, dt = s['case'], s['u'].dtype
    t, b, d = s['u'].shape
    frame, clip, valid = _order(s, t, b)

    def take(v):
        return torch.where(valid, v.float()[frame, clip], 0.)

    def give(v):
        return torch.where(valid, v, 0.)[frame, clip].to(dt)
    u, bm, cm, z = take(s['u']), take(s['b']), take(s['c']), take(s['z'])
    raw = take(s['delta']) + s['delta_bias']
    step = torch.where(valid, _softplus(raw), 0.)                           # 0 behind the last frame: the state stands still
    rate = -torch.exp(s['a_log'])
    decay = torch.exp(step[..., None] * rate)                               # [T, B, D, N]
    drive = (step * u)[..., None] * bm[:, :, None]
    if case['state']:
        drive[0] += decay[0] * s['ssm_state']
    h = _recurrence(decay, drive)
    del drive
    y = (h * cm[:, :, None]).sum(-1) + s['d'] * u
    sg = torch.sigmoid(z)
    out = give(y * z * sg)
    if not case['train']:
        return (out, h[-1].clone()) if case['state'] else out
    dy = take(s['dy'])
    dz = give(dy * y * sg * (1 + z * (1 - sg)))
    g = dy * z * sg
    r = g[..., None] * cm[:, :, None]
    r = _recurrence(torch.cat([torch.zeros_like(decay[:1]), decay[1:].flip(0)]), r.flip(0)).flip(0)
    dc = give((h * g[..., None]).sum(2))
    db = give((r * (step * u)[..., None]).sum(2))
    kept = r * decay * torch.cat([torch.zeros_like(h[:1]), h[:-1]]) * rate  # r[t] rate decay[t] h[t-1]
    del h, decay
    rb = (r * bm[:, :, None]).sum(-1)
    draw_ = (u * rb + kept.sum(-1)) * torch.sigmoid(raw)
    da = (kept * step[..., None]).sum((0, 1))
    return (out, give(g * s['d'] + step * rb), give(draw_), db, dc, dz, da, (g * u).sum((0, 1)),
            torch.where(valid, draw_, 0.).sum((0, 1)))


def _plain_step(s):
    dt = s['x'].dtype
    long = torch.cat([s['conv_state'].float(), s['x'].float()[:, None]], 1)
    pre = (long * s['weight'].t()).sum(1) + s['bias']
    step = _softplus(s['delta'].float() + s['delta_bias'])
    u, z = s['u'].float(), s['z'].float()
    h = torch.exp(step[..., None] * -torch.exp(s['a_log'])) * s['ssm_state'] + (step * u)[..., None] * s['b'].float()[:, None]
    y = ((h * s['c'].float()[:, None]).sum(-1) + s['d'] * u) * z * torch.sigmoid(z)
    return (pre * torch.sigmoid(pre)).to(dt), long[:, 1:].to(dt), y.to(dt), h


def _plain_norm(s):
    x, dy, dt = s['x'].float(), s['dy'].float(), s['x'].dtype
    c = x.shape[1]
    mean = x.sum(1, keepdim=True) / c
    xc = x - mean
    rstd = 1 / torch.sqrt((xc * xc).sum(1, keepdim=True) / c + 1e-5)
    xh = xc * rstd
    g = dy * s['weight']
    dx = rstd * (g - g.sum(1, keepdim=True) / c - xh * ((g * xh).sum(1, keepdim=True) / c))
    return (xh * s['weight'] + s['bias']).to(dt), dx.to(dt), (dy * xh).sum(0), dy.sum(0)


def _words(seed, step, site, n):
    """n 32-bit words of the counter-based generator Philox-4x32 with seven rounds (Salmon et al., SC 2011), as int64."""
    low = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, device=DEV)
    c = [block & low, block >> 32, torch.zeros_like(block) + (step & low), torch.full_like(block, site)]
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(7):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57                         # 32 x 32 -> 64 bits, modulo 2^64 as two's complement
        c = [((q >> 32) & low) ^ c[1] ^ k0, q & low, ((p >> 32) & low) ^ c[3] ^ k1, p & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack(c, 1).reshape(-1)[:n]


def _plain_dropout(s):
    x, p = s['x'], s['case']['p']
    keep = (_words(s['rng'][0], s['rng'][1], 3, x.numel()) >= int(p * 2 ** 32)).view(x.shape)
    y = torch.where(keep, x.float() * (1 / (1 - p)), 0.)
    if s['residual'] is not None:
        y = y + s['residual'].float()
    return y.to(x.dtype), torch.where(keep, s['dy'].float() * (1 / (1 - p)), 0.).to(x.dtype)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_conv(s):
    from pb_sed_amd import ops
    case = s['case']
    kw = dict(silu=True, seq_len=s['seq_len'], reverse=case['reverse'], state=s['conv_state'])
    y, state = ops.causal_conv_fwd(s['x'], s['weight'], s['bias'], want_state=not case['train'], **kw)
    if not case['train']:
        return y, state
    g = s['grads'].zero_()
    d, k = s['weight'].shape
    dw, db = g[:d * k].view(d, k), g[d * k:]
    dx, _ = ops.causal_conv_bwd(s['dy'], s['x'], s['weight'], s['bias'], dweight=dw, dbias=db, **kw)
    return y, dx, dw, db


def _own_scan(s):
    from pb_sed_amd import ops
    case = s['case']
    kw = dict(d=s['d'], z=s['z'], delta_bias=s['delta_bias'], softplus=True, seq_len=s['seq_len'], reverse=case['reverse'])
    args = s['u'], s['delta'], s['a_log'], s['b'], s['c']
    y, state, saved = ops.selective_scan_fwd(*args, state=s['ssm_state'], want_state=case['state'], save=case['train'], **kw)
    if not case['train']:
        return (y, state) if case['state'] else y
    g = s['grads'].zero_()
    d, n = s['a_log'].shape
    da, dd, dbias = g[:d * n].view(d, n), g[d * n:d * n + d], g[d * n + d:]
    du, ddelta, db, dc, dz, _ = ops.selective_scan_bwd(s['dy'], *args, saved, da_log=da, dd=dd, ddelta_bias=dbias, **kw)
    return y, du, ddelta, db, dc, dz, da, dd, dbias


def _own_step(s):
    from pb_sed_amd import ops
    x = ops.causal_conv_step(s['x'], s['weight'], s['bias'], s['conv_state'], silu=True, state_out=s['next_conv_state'])
    y = ops.selective_scan_step(s['u'], s['delta'], s['a_log'], s['b'], s['c'], s['ssm_state'], d=s['d'], z=s['z'],
                                delta_bias=s['delta_bias'], softplus=True, state_out=s['next_ssm_state'])
    return x, s['next_conv_state'], y, s['next_ssm_state']


def _own_norm(s):
    from pb_sed_amd import ops
    y, stats = ops.layer_norm_fwd(s['x'], s['weight'], s['bias'], eps=1e-5, save=True)
    g = s['grads'].zero_()
    dx = ops.layer_norm_bwd(s['dy'], s['x'], s['weight'], stats, dweight=g[0], dbias=g[1])
    return y, dx, g[0], g[1]


def _own_dropout(s):
    from pb_sed_amd import ops
    p = s['case']['p']
    return ops.dropout(s['x'], p, s['rng'], site=3, residual=s['residual']), ops.dropout(s['dy'], p, s['rng'], site=3)


def run(state):
    op = state['case']['op']
    if own:
        return {'conv': _own_conv, 'scan': _own_scan, 'step': _own_step, 'norm': _own_norm, 'dropout': _own_dropout}[op](state)
    return {'conv': _plain_conv, 'scan': _plain_scan, 'step': _plain_step, 'norm': _plain_norm, 'dropout': _plain_dropout}[op](state)


# ------------------------------------------------------------------------------------------------ work, definition
def work(case):
    """Each input read once, each output written once (frames behind a clip's end: outputs only); an exponential counts one."""
    e = torch.finfo(DTYPES[case['dtype']]).bits // 8
    op, train = case['op'], case['train']
    if op == 'norm':
        el = case['rows'] * case['c']
        return {'bytes': 4 * el * e + 16 * case['c'], 'flops': 22 * el}
    if op == 'dropout':
        el = case['rows'] * case['c']
        return {'bytes': (4 + case['residual']) * el * e, 'flops': (3 + case['residual']) * el}
    b, d = case['b'], case['d']
    if op == 'step':
        n, k = case['n'], case['k']
        return {'bytes': b * (2 * (k - 1) * d * e + 6 * d * e + 2 * n * e + 8 * d * n) + d * (4 * k + 4 * n + 12), 'flops': b * d * (2 * k + 8 * n + 20)}
    frames, valid = case['t'] * b, sum(lengths(case))
    if op == 'conv':
        k = case['k']
        moved = valid * d * e + frames * d * e + 4 * d * (k + 1) + (2 * b * (k - 1) * d * e if case['state'] else 0)
        ops_ = valid * d * (2 * k + 6)
        if train:                                     # x and dy in, dx, dw, db out
            moved += 2 * valid * d * e + frames * d * e + 8 * d * (k + 1)
            ops_ += valid * d * (6 * k + 14)
        return {'bytes': moved, 'flops': ops_}
    n = case['n']
    moved = valid * (3 * d + 2 * n) * e + frames * d * e + 4 * d * (n + 2) + (8 * b * d * n if case['state'] else 0)
    ops_ = valid * d * (7 * n + 20)
    if train:                                         # the inputs and dy again, five gradients of their sizes
        moved += valid * (4 * d + 2 * n) * e + frames * (3 * d + 2 * n) * e + 8 * d * (n + 2)
        ops_ += valid * d * (20 * n + 40)
    return {'bytes': moved, 'flops': ops_}


def exact(case, seed):
    s = prepare(case, seed)
    v = {key: x.double() for key, x in s.items() if isinstance(x, torch.Tensor) and x.is_floating_point()}
    return {'conv': _exact_conv, 'scan': _exact_scan, 'step': _exact_step, 'norm': _exact_norm, 'dropout': _exact_dropout}[case['op']](case, s, v)


def _frames(case, i, n):
    """The n frames of clip i in scan order."""
    return list(range(n))[::-1] if case['reverse'] else list(range(n))


def _exact_conv(case, s, v):
    t, b, d = v['x'].shape
    w, k = v['weight'], case['k']
    y, dx = torch.zeros_like(v['x']), torch.zeros_like(v['x'])
    dw, db = torch.zeros_like(w), torch.zeros_like(v['bias'])
    last = v['x'].new_zeros(b, k - 1, d)
    for i, n in enumerate(lengths(case)):
        x = v['x'][_frames(case, i, n), i]
        x = torch.cat([v['conv_state'][i] if case['state'] else x.new_zeros(k - 1, d), x])
        last[i] = x[n:]
        pre = v['bias'].repeat(n, 1)
        for j in range(k):
            pre += w[:, j] * x[j:j + n]
        e = torch.exp(-pre)
        y[_frames(case, i, n), i] = pre / (1 + e)
        if case['train']:
            g = v['dy'][_frames(case, i, n), i] * (1 / (1 + e) + pre * e / (1 + e) ** 2)
            gx = torch.zeros_like(x)
            for j in range(k):
                gx[j:j + n] += w[:, j] * g
                dw[:, j] += (g * x[j:j + n]).sum(0)
            db += g.sum(0)
            dx[_frames(case, i, n), i] = gx[k - 1:]
    return (y, dx, dw, db) if case['train'] else (y, last)


def _exact_scan(case, s, v):
    t, b, d = v['u'].shape
    lens, clip = torch.tensor(lengths(case), device=DEV), torch.arange(b, device=DEV)
    raw = v['delta'] + v['delta_bias']
    step = torch.where(raw > 0, raw + torch.log1p(torch.exp(-raw)), torch.log1p(torch.exp(raw)))
    rate = -torch.exp(v['a_log'])
    h = v['ssm_state'].clone() if case['state'] else v['u'].new_zeros(b, d, case['n'])
    out = {key: torch.zeros_like(v[src]) for key, src in (('y', 'u'), ('du', 'u'), ('dr', 'delta'), ('db', 'b'), ('dc', 'c'), ('dz', 'z'))}
    hs, ys = [], []
    gate = v['z'] / (1 + torch.exp(-v['z']))
    for p in range(t):
        f = (lens - 1 - p if case['reverse'] else torch.full_like(lens, p)).clamp_min(0)
        live = (p < lens).double()[:, None]
        st = step[f, clip] * live
        if case['train']:
            hs.append(h)
        h = torch.exp(st[..., None] * rate) * h + (st * v['u'][f, clip])[..., None] * v['b'][f, clip][:, None]
        y = (h * v['c'][f, clip][:, None]).sum(-1) + v['d'] * v['u'][f, clip]
        if case['train']:
            ys.append(y)
        out['y'].index_put_((f, clip), y * gate[f, clip] * live, accumulate=True)
    if not case['train']:
        return (out['y'], h) if case['state'] else out['y']
    da, dd, dbias, r = torch.zeros_like(rate), torch.zeros_like(v['d']), torch.zeros_like(v['d']), torch.zeros_like(h)
    for p in reversed(range(t)):
        f = (lens - 1 - p if case['reverse'] else torch.full_like(lens, p)).clamp_min(0)
        live = (p < lens).double()[:, None]
        u, z, st, dy = v['u'][f, clip], v['z'][f, clip], step[f, clip] * live, v['dy'][f, clip] * live
        sg = 1 / (1 + torch.exp(-z))
        g = dy * gate[f, clip]
        r = r + g[..., None] * v['c'][f, clip][:, None]
        decay = torch.exp(st[..., None] * rate)
        now = decay * hs[p] + (st * u)[..., None] * v['b'][f, clip][:, None]
        through = (r * decay * hs[p] * rate)
        rb = (r * v['b'][f, clip][:, None]).sum(-1)
        dr = (u * rb + through.sum(-1)) * live / (1 + torch.exp(-raw[f, clip]))
        for key, value in (('du', g * v['d'] + st * rb), ('dr', dr), ('db', (r * (st * u)[..., None]).sum(1)), ('dc', (now * g[..., None]).sum(1)),
                           ('dz', dy * ys[p] * sg * (1 + z * (1 - sg)))):
            out[key].index_put_((f, clip), value, accumulate=True)
        da += (through * st[..., None]).sum(0)
        dd += (g * u).sum(0)
        dbias += dr.sum(0)
        r = r * decay
    return out['y'], out['du'], out['dr'], out['db'], out['dc'], out['dz'], da, dd, dbias


def _exact_step(case, s, v):
    pre = v['bias'] + v['x'] * v['weight'][:, -1]
    for j in range(case['k'] - 1):
        pre = pre + v['conv_state'][:, j] * v['weight'][:, j]
    kept = torch.cat([v['conv_state'][:, 1:], v['x'][:, None]], 1)
    step = torch.logaddexp(v['delta'] + v['delta_bias'], torch.zeros_like(v['delta']))
    h = v['ssm_state'] * torch.exp(-torch.exp(v['a_log']) * step[..., None]) + torch.einsum('bd,bn->bdn', step * v['u'], v['b'])
    y = torch.einsum('bdn,bn->bd', h, v['c']) + v['u'] * v['d']
    return pre / (1 + torch.exp(-pre)), kept, y * v['z'] / (1 + torch.exp(-v['z'])), h


def _exact_norm(case, s, v):
    mean, var = v['x'].mean(1, keepdim=True), v['x'].var(1, unbiased=False, keepdim=True)
    std = (var + 1e-5).sqrt()
    xh = (v['x'] - mean) / std
    g = v['dy'] * v['weight']
    dx = (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True)) / std
    return xh * v['weight'] + v['bias'], dx, torch.einsum('rc,rc->c', v['dy'], xh), v['dy'].sum(0)


def _exact_dropout(case, s, v):
    import numpy as np
    seed, step = (int(x) for x in s['rng'].tolist())
    n = v['x'].numel()
    i = np.arange(0, n, 4, dtype=np.uint64) >> np.uint64(2)
    u32, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    x0, x1, x2, x3 = i & u32, i >> half, np.full_like(i, step & 0xFFFFFFFF), np.full_like(i, 3)
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(7):
        a, b = x0 * np.uint64(0xD2511F53), x2 * np.uint64(0xCD9E8D57)
        x0, x1, x2, x3 = (b >> half) ^ x1 ^ np.uint64(key[0]), b & u32, (a >> half) ^ x3 ^ np.uint64(key[1]), a & u32
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    words = np.stack([x0, x1, x2, x3], 1).reshape(-1)[:n]
    keep = torch.from_numpy(words >= np.uint64(int(case['p'] * 2 ** 32))).to(DEV).view(v['x'].shape).double()
    y = v['x'] * keep / (1 - case['p'])
    return (y + v['residual'] if case['residual'] else y), v['dy'] * keep / (1 - case['p'])
