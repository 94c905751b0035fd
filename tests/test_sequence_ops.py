"""The state-space sequence operators of pb_sed_amd.ops (causal_conv_*, selective_scan_*, layer_norm_*, dropout) against the float64
restatements of tests/sequence_ref.py: on the GPU, and - the same kernel sources compiled for the host (tests/emu) - on the CPU, where
uninitialised memory is NaN.  The bounds are derived in tests/sequence_ref.py; the factors k below count roundings per term."""
import contextlib
import ctypes
import itertools

import numpy as np
import pytest
import torch

from tests import sequence_ref as ref
from tests.sequence_ref import check

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope='module')
def emulated_library(tmp_path_factory):
    from tests.emu import cpu_device

    class Library(cpu_device.EmulatedLibrary):
        def __init__(self, path):
            self._units, self._fns, self._last, self.calls, self.seconds = {'sequence': ctypes.CDLL(path)}, {}, 'sequence', [], {}
    return Library(cpu_device.compile_unit('sequence', cpu_device.os.path.join(cpu_device.ROOT, 'pb_sed_amd', 'csrc'),
                                           str(tmp_path_factory.mktemp('sequence') / 'libemu_sequence.so')))


@pytest.fixture(params=['emulated', pytest.param('cuda', marks=pytest.mark.gpu)])
def dev(request, monkeypatch):
    if request.param == 'cuda':
        yield 'cuda:0'
        return
    from tests.emu import cpu_device
    with cpu_device.emulated_device(monkeypatch, request.getfixturevalue('emulated_library')):
        yield 'cpu'


def normal(g, *shape, scale=1.):
    return torch.randn(*shape, generator=g, dtype=torch.float64) * scale


def rounded(v, dtype):
    """(the tensor in its type, the same values in float64)"""
    v = v.to(dtype)
    return v, v.double()


def slot(v, dev, pad=3, strided=True):
    """``v`` [..., C] on the device inside a wider buffer filled with NaN: odd offsets, a row stride that no vector length divides."""
    if not strided:
        return v.to(dev)
    wide = torch.full((*v.shape[:-1], v.shape[-1] + 2 * pad + 1), float('nan'), dtype=v.dtype)
    wide[..., pad:pad + v.shape[-1]] = v
    return wide.to(dev)[..., pad:pad + v.shape[-1]]


def poison(v, seq_len, value=float('nan')):
    """Frames behind the clips' ends become ``value`` (they must not be read)."""
    if seq_len is not None:
        for i, n in enumerate(seq_len):
            v[int(n):, i] = value
    return v


def lens(seq_len, dev):
    return None if seq_len is None else torch.tensor(seq_len, dtype=torch.int32).to(dev)


# ------------------------------------------------------------------------------------------------ causal convolution
CONV = [  # t, b, d, k, seq_len, reverse, state, silu, bias, dtype
    (1, 1, 1, 2, None, False, True, True, True, F32),
    (1, 3, 5, 4, [1, 0, 1], True, True, True, True, BF16),
    (2, 2, 8, 8, [2, 1], False, True, False, False, F32),            # fewer frames than taps
    (23, 3, 13, 4, [23, 0, 7], False, False, True, True, F32),
    (23, 3, 13, 4, [23, 0, 7], True, True, True, False, F16),
    (70, 2, 36, 3, [70, 64], False, True, True, True, BF16),          # several load groups, runs that meet
    (70, 2, 36, 5, None, True, False, True, True, F32),
    (37, 1, 300, 2, None, False, False, False, True, F32),           # more than one channel group
]


@pytest.mark.parametrize('case', CONV, ids=lambda c: '-'.join(str(v) for v in c).replace(' ', ''))
@pytest.mark.parametrize('strided', [False, True])
def test_causal_conv_forward_and_gradients(dev, case, strided):
    from pb_sed_amd import ops
    t, b, d, k, seq_len, reverse, with_state, silu, with_bias, dtype = case
    g = torch.Generator().manual_seed(t * 131 + d)
    x, x64 = rounded(normal(g, t, b, d), dtype)
    dy, dy64 = rounded(normal(g, t, b, d), dtype)
    w, w64 = rounded(normal(g, d, k, scale=k ** -.5), F32)
    bias, bias64 = rounded(normal(g, d), F32) if with_bias else (None, None)
    state, state64 = rounded(normal(g, b, k - 1, d), dtype) if with_state else (None, None)
    ds, ds64 = rounded(normal(g, b, k - 1, d), dtype) if with_state else (None, None)
    want = ref.conv(x64, w64, bias64, silu=silu, seq_len=seq_len, reverse=reverse, state=state64, dy=dy64, dstate_out=ds64)
    up = lambda v: None if v is None else v.to(dev)                      # noqa: E731
    kw = dict(silu=silu, seq_len=lens(seq_len, dev), reverse=reverse, state=up(state))
    xd, gd = slot(poison(x, seq_len), dev, strided=strided), slot(poison(dy, seq_len), dev, strided=strided)
    y, state_out = ops.causal_conv_fwd(xd, up(w), up(bias), want_state=True, **kw)
    check(y, want['y'], want['major']['y'], k + 10, 'y')
    assert torch.equal(state_out.cpu().double(), want['state_out'])       # copies of the inputs
    dw, db = torch.full((d, k), .5, device=dev), torch.full((d,), -2., device=dev)
    out = slot(torch.zeros(t, b, d, dtype=dtype), dev) if strided else None
    dx, dstate = ops.causal_conv_bwd(gd, xd, up(w), up(bias), dweight=dw, dbias=db if with_bias else None, dstate_out=up(ds), want_dstate=True,
                                     dx=out, **kw)
    assert out is None or dx is out
    check(dx, want['dx'], want['major']['dx'], 2 * k + 14, 'dx')
    check(dstate, want['dstate'], want['major']['dstate'], 2 * k + 14, 'dstate')
    sums = 2 * k + 14 + 64 + 4                                            # a run's 64 terms, a block's four runs; the rest in double
    check(dw, want['dw'] + .5, want['major']['dw'] + .5, sums, 'dweight')
    if with_bias:
        check(db, want['db'] - 2, want['major']['db'] + 2, sums, 'dbias')
    else:
        assert (db == -2).all()


def test_causal_conv_pieces_and_single_frames_follow_the_whole(dev):
    """A recording cut into pieces with carried states, and frame by frame, gives the bits of one call."""
    from pb_sed_amd import ops
    g = torch.Generator().manual_seed(3)
    for dtype, k in itertools.product((F32, BF16), (2, 4, 8)):
        x = normal(g, 21, 2, 9).to(dtype).to(dev)
        w, bias = normal(g, 9, k).float().to(dev), normal(g, 9).float().to(dev)
        whole, last = ops.causal_conv_fwd(x, w, bias, want_state=True)
        y0, s0 = ops.causal_conv_fwd(x[:13], w, bias, want_state=True)
        y1, s1 = ops.causal_conv_fwd(x[13:], w, bias, state=s0, want_state=True)
        assert torch.equal(torch.cat([y0, y1]), whole) and torch.equal(s1, last)
        state = torch.zeros(2, k - 1, 9, dtype=dtype, device=dev)
        other = torch.empty_like(state)
        for f in range(21):
            if f % 2:
                y = ops.causal_conv_step(x[f], w, bias, state, state_out=other)
                state, other = other, state
            else:
                y = ops.causal_conv_step(x[f], w, bias, state)            # in place
            assert torch.equal(y, whole[f]), (dtype, k, f)
        assert torch.equal(state, last)


# ------------------------------------------------------------------------------------------------ selective scan
def scan_inputs(g, t, b, d, n, dtype, full=True, state=False):
    v = dict(u=rounded(normal(g, t, b, d), dtype), delta=rounded(normal(g, t, b, d, scale=.7), dtype), b=rounded(normal(g, t, b, n), dtype),
             c=rounded(normal(g, t, b, n), dtype), a_log=rounded(normal(g, d, n, scale=1.), F32), dy=rounded(normal(g, t, b, d), dtype))
    if full:
        v.update(z=rounded(normal(g, t, b, d), dtype), d=rounded(normal(g, d), F32), delta_bias=rounded(normal(g, d) - 2, F32))
    if state:
        v.update(state=rounded(normal(g, b, d, n), F32), dstate_out=rounded(normal(g, b, d, n), F32))
    return {key: x for key, (x, _) in v.items()}, {key: x for key, (_, x) in v.items()}


SCAN = [  # t, b, d, n, seq_len, reverse, everything optional given, state, softplus, dtype
    (1, 1, 1, 1, None, False, True, True, True, F32),
    (1, 2, 3, 5, [1, 0], True, False, True, True, BF16),
    (7, 2, 65, 8, [7, 3], False, True, False, True, F32),             # a channel block and one channel; a part of a tile
    (16, 1, 33, 16, None, True, True, True, True, F16),
    (33, 3, 9, 12, [33, 0, 17], True, True, True, True, F32),
    (50, 2, 40, 16, [50, 32], False, True, False, True, BF16),
    (35, 2, 10, 20, [34, 35], True, False, True, False, F32),         # no softplus: the sum itself, also below zero
    (66, 1, 5, 33, None, False, True, True, True, F32),
    (70, 1, 4, 64, [65], True, True, False, True, F32),
    (300, 1, 9, 16, [289], False, True, True, True, F32),             # cut into runs
    (260, 2, 3, 3, [260, 100], True, True, True, True, F32),
    (1100, 1, 3, 2, None, True, True, True, True, F32),               # many runs: their states are folded by a launch of their own
]


@pytest.mark.parametrize('case', SCAN, ids=lambda c: '-'.join(str(v) for v in c).replace(' ', ''))
@pytest.mark.parametrize('strided', [False, True])
def test_selective_scan_forward_and_gradients(dev, case, strided):
    from pb_sed_amd import ops
    t, b, d, n, seq_len, reverse, full, with_state, softplus, dtype = case
    g = torch.Generator().manual_seed(t * 17 + n)
    v, v64 = scan_inputs(g, t, b, d, n, dtype, full, with_state)
    if not softplus:
        v['delta'], v64['delta'] = rounded(v64['delta'] * .2, dtype)
    keys = ('d', 'z', 'delta_bias', 'state')
    want = ref.scan(*(v64[key] for key in ('u', 'delta', 'a_log', 'b', 'c')), softplus=softplus, seq_len=seq_len, reverse=reverse, dy=v64['dy'],
                    dstate_out=v64.get('dstate_out'), **{key: v64.get(key) for key in keys})
    major = want['major']
    frames = ('u', 'delta', 'b', 'c', 'z', 'dy')
    dv = {key: slot(poison(x, seq_len), dev, strided=strided) if key in frames else x.to(dev) for key, x in v.items()}
    args = [dv[key] for key in ('u', 'delta', 'a_log', 'b', 'c')]
    kw = dict(d=dv.get('d'), z=dv.get('z'), delta_bias=dv.get('delta_bias'), softplus=softplus, seq_len=lens(seq_len, dev), reverse=reverse)
    y, state_out, saved = ops.selective_scan_fwd(*args, state=dv.get('state'), want_state=True, save=True, **kw)
    # 20 roundings of a state per frame (softplus 12, rate 3, exponential 2, products and sum 3; their propagation is in the majorant),
    # 10 of y behind it; cut into runs: sums of D over at most 64 frames more
    k = 30 + (64 if t > 64 else 0)
    check(y, want['y'], major['y'], k, 'y')
    check(state_out, want['state_out'], major['state_out'], k, 'state_out')
    again, _, none = ops.selective_scan_fwd(*args, state=dv.get('state'), **kw)
    assert none is None and torch.equal(again, y)
    da, dd, dbias = torch.full((d, n), 1.5, device=dev), torch.full((d,), -.5, device=dev), torch.full((d,), 3., device=dev)
    out = slot(torch.zeros(t, b, d, dtype=dtype), dev) if strided and full else None
    du, ddelta, db, dc, dz, dstate = ops.selective_scan_bwd(
        dv['dy'], *args, saved, da_log=da, dd=dd if full else None, ddelta_bias=dbias if full else None, dstate_out=dv.get('dstate_out'),
        want_dstate=True, dz=out, **kw)
    # states and adjoints carry k each; a sum over the channels adds 16 + channel blocks, one over frames 16 + tiles (then double)
    k = 2 * k + 20 + 16 + t // 16
    for key, got in (('du', du), ('ddelta', ddelta), ('db', db), ('dc', dc), ('dstate', dstate)):
        check(got, want[key], major[key], k, key)
    check(da, want['da_log'] + 1.5, major['da_log'] + 1.5, k, 'da_log')
    if full:
        assert out is None or dz is out
        check(dz, want['dz'], major['dz'], k, 'dz')
        check(dd, want['dd'] - .5, major['dd'] + .5, k, 'dd')
        check(dbias, want['ddelta_bias'] + 3, major['ddelta_bias'] + 3, k, 'ddelta_bias')
    else:
        assert dz is None


def test_scan_formulas_against_differences():
    """The gradients that the kernels are compared with, against central differences of the forward formula in float64."""
    g = torch.Generator().manual_seed(0)
    _, v = scan_inputs(g, 6, 2, 3, 2, F32, True, True)
    seq_len = [6, 4]
    keys = dict(u='du', delta='ddelta', b='db', c='dc', z='dz', a_log='da_log', d='dd', delta_bias='ddelta_bias', state='dstate')

    def loss(**over):
        o = {**v, **over}
        r = ref.scan(o['u'], o['delta'], o['a_log'], o['b'], o['c'], d=o['d'], z=o['z'], delta_bias=o['delta_bias'], state=o['state'], seq_len=seq_len,
                     reverse=True)
        return float((r['y'] * v['dy']).sum() + (r['state_out'] * v['dstate_out']).sum())
    grads = ref.scan(v['u'], v['delta'], v['a_log'], v['b'], v['c'], d=v['d'], z=v['z'], delta_bias=v['delta_bias'], state=v['state'], seq_len=seq_len,
                     reverse=True, dy=v['dy'], dstate_out=v['dstate_out'])
    for key, grad in keys.items():
        for _ in range(4):
            e = torch.randn(v[key].shape, generator=g, dtype=torch.float64)
            h = 1e-6
            diff = (loss(**{key: v[key] + h * e}) - loss(**{key: v[key] - h * e})) / (2 * h)
            # the differences' own error: h^2 third derivatives and 1e-16 / h of a loss of order 10
            assert abs(diff - float((grads[grad] * e).sum())) < 1e-7 * (1 + abs(diff)), key


def test_conv_and_norm_formulas_against_differences():
    g = torch.Generator().manual_seed(1)
    x, w, bias, state, dy, ds = (normal(g, *s) for s in ((7, 2, 3), (3, 4), (3,), (2, 3, 3), (7, 2, 3), (2, 3, 3)))
    kw = dict(seq_len=[7, 2], reverse=True)
    grads = ref.conv(x, w, bias, state=state, dy=dy, dstate_out=ds, **kw)

    def loss(x, w, bias, state):
        r = ref.conv(x, w, bias, state=state, **kw)
        return float((r['y'] * dy).sum() + (r['state_out'] * ds).sum())
    for i, name in enumerate(('dx', 'dw', 'db', 'dstate')):
        args = [x, w, bias, state]
        e = normal(g, *args[i].shape)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + 1e-6 * e, args[i] - 1e-6 * e
        diff = (loss(*up) - loss(*down)) / 2e-6
        assert abs(diff - float((grads[name] * e).sum())) < 1e-7 * (1 + abs(diff)), name
    x, w, b, dy = (normal(g, *s) for s in ((5, 7), (7,), (7,), (5, 7)))
    grads = ref.layer_norm(x, w, b, 1e-5, dy)
    for i, name in enumerate(('dx', 'dw', 'db')):
        args = [x, w, b]
        e = normal(g, *args[i].shape)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + 1e-6 * e, args[i] - 1e-6 * e
        diff = float(((ref.layer_norm(*up, 1e-5)['y'] - ref.layer_norm(*down, 1e-5)['y']) * dy).sum()) / 2e-6
        assert abs(diff - float((grads[name] * e).sum())) < 1e-6 * (1 + abs(diff)), name


@pytest.mark.parametrize('n', [3, 8, 16, 30, 64])
@pytest.mark.parametrize('dtype', [F32, F16])
def test_selective_scan_single_frames(dev, n, dtype):
    """One frame of several streams, in place and into another buffer, against the restatement."""
    from pb_sed_amd import ops
    g = torch.Generator().manual_seed(n)
    b, d = 5, 70
    v, v64 = scan_inputs(g, 1, b, d, n, dtype, True, True)
    want = ref.scan(*(v64[key] for key in ('u', 'delta', 'a_log', 'b', 'c')), **{key: v64[key] for key in ('d', 'z', 'delta_bias', 'state')})
    one = {key: slot(v[key][0], dev) for key in ('u', 'delta', 'b', 'c', 'z')}
    par = {key: v[key].to(dev) for key in ('a_log', 'd', 'delta_bias')}
    state, other = v['state'].to(dev), torch.empty_like(v['state']).to(dev)
    args = one['u'], one['delta'], par['a_log'], one['b'], one['c'], state
    kw = dict(d=par['d'], z=one['z'], delta_bias=par['delta_bias'])
    y = ops.selective_scan_step(*args, state_out=other, **kw)
    assert torch.equal(state.cpu(), v['state'])
    check(y, want['y'][0], want['major']['y'][0], 30 + n, 'y')
    check(other, want['state_out'], want['major']['state_out'], 20, 'state')
    again = ops.selective_scan_step(*args, **kw)
    assert torch.equal(again, y) and torch.equal(state, other)
    bare = ops.selective_scan_step(one['u'], one['delta'], par['a_log'], one['b'], one['c'], v['state'].to(dev), softplus=False)
    want = ref.scan(*(v64[key] for key in ('u', 'delta', 'a_log', 'b', 'c')), softplus=False, state=v64['state'])
    check(bare, want['y'][0], want['major']['y'][0], 30 + n, 'y, nothing optional')


def test_selective_scan_pieces_follow_the_whole(dev):
    from pb_sed_amd import ops
    g = torch.Generator().manual_seed(9)
    v, v64 = scan_inputs(g, 45, 2, 20, 16, F32)
    x = {key: t.to(dev) for key, t in v.items()}

    def run(a, b, state):
        cut = {key: x[key][a:b] for key in ('u', 'delta', 'b', 'c', 'z')}
        return ops.selective_scan_fwd(cut['u'], cut['delta'], x['a_log'], cut['b'], cut['c'], d=x['d'], z=cut['z'], delta_bias=x['delta_bias'], state=state,
                                      want_state=True)[:2]
    want = ref.scan(*(v64[key] for key in ('u', 'delta', 'a_log', 'b', 'c')), **{key: v64[key] for key in ('d', 'z', 'delta_bias')})
    y0, s0 = run(0, 16, None)
    y1, s1 = run(16, 17, s0)
    y2, s2 = run(17, 45, s1)
    check(torch.cat([y0, y1, y2]), want['y'], want['major']['y'], 30, 'y')
    check(s2, want['state_out'], want['major']['state_out'], 30, 'state')


def test_selective_scan_extreme_values(dev):
    """Steps that forget everything, steps of zero, rates beyond float32: finite where the formula is; NaN stays in its channel and clip
    (b, c: in its clip), and in the frames behind it."""
    from pb_sed_amd import ops
    t, b, d, n = 20, 2, 10, 4
    g = torch.Generator().manual_seed(2)
    u, delta, bm, cm = (normal(g, t, b, k).float() for k in (d, d, n, n))
    a_log = torch.zeros(d, n)
    a_log[:, 1], a_log[:, 2], a_log[:, 3] = 200., -200., 20.              # rates inf, 0, 5e8
    delta[:, :, 3], delta[:, :, 4], delta[:, :, 5] = 300., -300., -60.    # D = 300, 0, 9e-27
    seq_len = torch.tensor([20, 11], dtype=torch.int32).to(dev)
    run = lambda u, bm: ops.selective_scan_fwd(u.to(dev), delta.to(dev), a_log.to(dev), bm.to(dev), cm.to(dev), seq_len=seq_len, want_state=True)[:2]     # noqa: E731
    y, h = run(u, bm)
    assert torch.isfinite(y).all() and torch.isfinite(h).all()
    bad = u.clone()
    bad[6, 0, 2] = float('nan')
    y2, h2 = run(bad, bm)
    nan = torch.isnan(y2.cpu())
    assert nan[6:, 0, 2].all() and nan.sum() == 14
    assert torch.equal(y2[~torch.isnan(y2)], y[~torch.isnan(y2)])
    worse = bm.clone()
    worse[5, 1, 0] = float('inf')
    y3, _ = run(u, worse)
    assert torch.equal(y3[:, 0], y[:, 0]) and torch.equal(y3[:5, 1], y[:5, 1]) and not torch.isfinite(y3[5:11, 1, :3].cpu()).any()
    assert (y3[11:, 1] == 0).all()


# ------------------------------------------------------------------------------------------------ layer norm
NORM = [  # rows, C
    ((3,), 1), ((1,), 2), ((5, 3), 7), ((2, 2, 3), 8), ((9,), 17), ((70,), 64), ((5,), 65), ((4,), 257), ((3,), 513), ((6,), 1023), ((2,), 1024),
    ((2,), 1500), ((2,), 2049), ((1,), 4100), ((3,), 8195)]


@pytest.mark.parametrize('lead,c', NORM, ids=lambda v: str(v).replace(' ', ''))
@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('strided,affine', [(False, True), (True, False), (True, True)])
def test_layer_norm_forward_and_gradients(dev, lead, c, dtype, strided, affine):
    from pb_sed_amd import ops
    g = torch.Generator().manual_seed(c)
    x, x64 = rounded(normal(g, *lead, c) * 3 + 5 * normal(g, *lead, 1), dtype)
    dy, dy64 = rounded(normal(g, *lead, c), dtype)
    w, w64 = rounded(normal(g, c), F32) if affine else (None, None)
    b, b64 = rounded(normal(g, c), F32) if affine else (None, None)
    want = ref.layer_norm(x64, w64, b64, 1e-3, dy64)
    up = lambda v: None if v is None else v.to(dev)                       # noqa: E731
    xd, gd = slot(x, dev, strided=strided), slot(dy, dev, strided=strided)
    y, stats = ops.layer_norm_fwd(xd, up(w), up(b), eps=1e-3, save=True)
    sums = 33 + 9                                                         # a lane's values one after the other, then the lanes' tree
    check(y, want['y'], want['major']['y'], 2 * sums + 8, 'y')
    plain, none = ops.layer_norm_fwd(xd, up(w), up(b), eps=1e-3)
    assert none is None and torch.equal(plain, y)
    dw, db = torch.full((c,), 1., device=dev), torch.full((c,), -1., device=dev)
    dx = ops.layer_norm_bwd(gd, xd, up(w), stats, dweight=dw, dbias=db)
    rows = int(np.prod(lead))
    check(dx, want['dx'], want['major']['dx'], 4 * sums + 20, 'dx')
    check(dw, want['dw'] + 1, want['major']['dw'] + 1, 2 * sums + 8 + rows, 'dweight')
    check(db, want['db'] - 1, want['major']['db'] + 1, rows + 8, 'dbias')
    assert torch.equal(ops.layer_norm_bwd(gd, xd, up(w), stats), dx)      # without the weights' gradients


def test_layer_norm_rows_do_not_mix(dev):
    from pb_sed_amd import ops
    for c in (10, 300, 9000):
        x = torch.randn(6, c, generator=torch.Generator().manual_seed(c))
        x[2, c // 2] = float('nan')
        x[4] = 7.                                                         # no variance
        y, _ = ops.layer_norm_fwd(x.to(dev), eps=1e-5)
        y = y.cpu()
        assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3, 4, 5]]).all() and (y[4].abs() < 1e-2).all()


# ------------------------------------------------------------------------------------------------ dropout
def test_generator_matches_the_published_vectors():
    """Known answers of Philox-4x32 for counter and key zero: ten and seven rounds."""
    assert [hex(int(v)) for v in ref.philox_words(0, 0, 0, 4, 10)] == ['0x6627e8d5', '0xe169c58d', '0xbc57ac4c', '0x9b00dbd8']
    assert [hex(int(v)) for v in ref.philox_words(0, 0, 0, 4, 7)] == ['0x5f6fb709', '0xd893f64', '0x4f121f81', '0x4f730a48']


@pytest.mark.parametrize('shape', [(1, 1), (3, 7), (5, 8), (2, 3, 12), (33, 20), (1, 2050)], ids=str)
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('p', [0., .1, .5, 1.])
def test_dropout_mask_is_the_generators(dev, shape, dtype, p):
    from pb_sed_amd import ops
    n = int(np.prod(shape))
    seed, step, site = 0x123456789ABCDEF, (5 << 32) + 0xFFFFFFFE, 11          # the step counts modulo 2^32
    keep = torch.from_numpy(ref.philox_words(seed, step, site, n) >= np.uint64(int(p * 2 ** 32))).view(shape) & (p < 1)
    g = torch.Generator().manual_seed(n)
    x, x64 = rounded(normal(g, *shape), dtype)
    res, res64 = rounded(normal(g, *shape), dtype)
    rng = torch.tensor([seed, step]).to(dev)
    want = torch.where(keep, x64 / (1 - p if p < 1 else 1), 0.)
    for strided in (False, True):
        xd, rd = slot(x, dev, strided=strided), slot(res, dev, strided=strided)
        y = ops.dropout(xd, p, rng, site=site)
        check(y, want, want.abs(), 2, 'y')
        z = ops.dropout(xd, p, rng, site=site, residual=rd)
        check(z, want + res64, want.abs() + res64.abs(), 3, 'with a residual')
        out = slot(torch.zeros(shape, dtype=dtype), dev) if strided else torch.empty(shape, dtype=dtype, device=dev)
        assert ops.dropout(xd, p, rng, site=site, residual=rd, out=out) is out and torch.equal(out, z)
        inplace = slot(x, dev, strided=strided)
        ops.dropout(inplace, p, rng, site=site, out=inplace)
        assert torch.equal(inplace, y)
        target = slot(res, dev, strided=strided)
        ops.dropout(xd, p, rng, site=site, residual=target, out=target)
        assert torch.equal(target, z)


def test_dropout_drops_by_selection_and_draws_anew(dev):
    from pb_sed_amd import ops
    rng = torch.tensor([77, 0]).to(dev)
    x = torch.full((40, 25), float('inf'))
    y = ops.dropout(x.to(dev), .5, rng).cpu()
    assert ((y == 0) | (y == float('inf'))).all() and (y == 0).any()       # no 0 x inf
    ones = torch.ones(40, 25).to(dev)
    masks = [ops.dropout(ones, .5, rng, site=s) for s in (0, 1)]
    rng[1] += 1
    masks.append(ops.dropout(ones, .5, rng))
    rng[0] += 1
    masks.append(ops.dropout(ones, .5, rng))
    for a, b in itertools.combinations(masks, 2):
        agree = float((a == b).float().mean())
        assert abs(agree - .5) < 5 * .5 / 1000 ** .5, agree               # 1000 fair coins, five standard deviations
    for m in masks:
        assert abs(float((m == 2).float().mean()) - .5) < 5 * .5 / 1000 ** .5


# ------------------------------------------------------------------------------------------------ refusals (no kernel runs)
def test_refusals(dev):
    from pb_sed_amd import ops
    f = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype, device=dev)     # noqa: E731
    x, w, st = f(4, 2, 6), f(6, 3), f(2, 2, 6)
    rng = torch.zeros(2, dtype=torch.int64, device=dev)
    u, al, bc = f(4, 2, 6), f(6, 5), f(4, 2, 5)
    scan = lambda **k: ops.selective_scan_fwd(**{**dict(u=u, delta=u, a_log=al, b=bc, c=bc), **k})        # noqa: E731
    y, _, saved = scan(save=True)
    bwd = lambda **k: ops.selective_scan_bwd(**{**dict(dy=u, u=u, delta=u, a_log=al, b=bc, c=bc, saved=saved), **k})      # noqa: E731
    step = lambda **k: ops.selective_scan_step(**{**dict(u=u[0], delta=u[0], a_log=al, b=bc[0], c=bc[0], state=f(2, 6, 5)), **k})     # noqa: E731
    long = f(2 * 2 * 6 + 6)
    refused = [
        lambda: ops.causal_conv_fwd(f(4, 2, 6, dtype=torch.float64), w), lambda: ops.causal_conv_fwd(f(4, 6), w),
        lambda: ops.causal_conv_fwd(f(0, 2, 6), w), lambda: ops.causal_conv_fwd(x, f(6, 1)), lambda: ops.causal_conv_fwd(x, f(6, 9)),
        lambda: ops.causal_conv_fwd(x, f(5, 3)), lambda: ops.causal_conv_fwd(x, w.to(BF16)), lambda: ops.causal_conv_fwd(x, f(3, 6).t()),
        lambda: ops.causal_conv_fwd(x, w, f(5)), lambda: ops.causal_conv_fwd(x, w, seq_len=f(2)), lambda: ops.causal_conv_fwd(f(4, 6, 2).transpose(1, 2), w),
        lambda: ops.causal_conv_fwd(x, w, seq_len=torch.zeros(3, dtype=torch.int32, device=dev)), lambda: ops.causal_conv_fwd(x, w, state=f(2, 3, 6)),
        lambda: ops.causal_conv_fwd(x, w, state=st.to(BF16)), lambda: ops.causal_conv_bwd(x.to(F16), x, w), lambda: ops.causal_conv_bwd(None, x, w),
        lambda: ops.causal_conv_bwd(x, x, w, dx=x), lambda: ops.causal_conv_bwd(x.clone(), x, w, dx=x[:1].expand(4, 2, 6)),
        lambda: ops.causal_conv_bwd(x, x, w, dweight=f(6, 2)), lambda: ops.causal_conv_step(x, w, None, st), lambda: ops.causal_conv_step(x[0], w, None, None),
        lambda: ops.causal_conv_step(f(2, 6), w, None, long[:24].view(2, 2, 6), state_out=long[6:30].view(2, 2, 6)),
        lambda: scan(u=f(2, 6)), lambda: scan(delta=f(4, 2, 5)), lambda: scan(a_log=f(6, 65), b=f(4, 2, 65), c=f(4, 2, 65)), lambda: scan(a_log=f(5, 5)),
        lambda: scan(b=f(4, 2, 6)), lambda: scan(c=None), lambda: scan(d=f(5)), lambda: scan(z=u.to(BF16)), lambda: scan(state=f(2, 6, 4)),
        lambda: scan(seq_len=torch.zeros(2, dtype=torch.int64, device=dev)), lambda: scan(u=f(4, 6, 2).transpose(1, 2)), lambda: scan(state=f(2, 6, 5, dtype=F16)),
        lambda: bwd(saved=None), lambda: bwd(saved=f(3)), lambda: bwd(dz=f(4, 2, 6)), lambda: bwd(z=u, dz=u), lambda: bwd(da_log=f(6, 4)), lambda: bwd(dy=None),
        lambda: bwd(z=u.clone(), dz=f(1, 2, 6).expand(4, 2, 6)), lambda: bwd(dstate_out=f(2, 6)),
        lambda: step(u=u), lambda: step(state=None), lambda: step(state=f(2, 6, 5, dtype=BF16)), lambda: step(b=bc[0, :, :4]), lambda: step(z=f(2, 5)),
        lambda: ops.layer_norm_fwd(f(3, 0)), lambda: ops.layer_norm_fwd(x, f(5)), lambda: ops.layer_norm_fwd(x, eps=-1.), lambda: ops.layer_norm_fwd(x, eps=float('nan')),
        lambda: ops.layer_norm_fwd(f(4, 6, 2).transpose(1, 2)), lambda: ops.layer_norm_fwd(f(4, 3, 6)[:, :2]), lambda: ops.layer_norm_fwd(f(1, 6).expand(4, 6)),
        lambda: ops.layer_norm_bwd(x, x, None, None), lambda: ops.layer_norm_bwd(x, x, None, f(7, 2)), lambda: ops.layer_norm_bwd(f(4, 2, 5), x, None, f(8, 2)),
        lambda: ops.dropout(x, -.1, rng), lambda: ops.dropout(x, 1.1, rng), lambda: ops.dropout(x, float('nan'), rng), lambda: ops.dropout(x, .1, rng.int()),
        lambda: ops.dropout(x, .1, None), lambda: ops.dropout(x, .1, rng, site=-1), lambda: ops.dropout(x, .1, rng, site=1 << 31),
        lambda: ops.dropout(x, .1, rng, residual=f(4, 2, 5)), lambda: ops.dropout(x, .1, rng, out=f(4, 6, 2).transpose(1, 2)),
        lambda: ops.dropout(long[:24].view(4, 6), .1, rng, out=long[6:30].view(4, 6)), lambda: ops.dropout(f(24).view(4, 6), .1, rng, out=f(1, 6).expand(4, 6)),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f'call {i} was accepted')


def test_sums_that_share_memory_are_refused(dev):
    from pb_sed_amd import ops
    f = lambda *s: torch.zeros(*s, device=dev)     # noqa: E731
    x, w, a_log, bc, both = f(4, 2, 6), f(6, 3), f(6, 1), f(4, 2, 1), f(30)
    saved = ops.selective_scan_fwd(x, x, a_log, bc, bc, save=True)[2]
    stats = ops.layer_norm_fwd(x, save=True)[1]
    for call in (lambda: ops.causal_conv_bwd(x, x, w, dweight=both[:18].view(6, 3), dbias=both[17:23]),
                 lambda: ops.selective_scan_bwd(x, x, x, a_log, bc, bc, saved, da_log=both[:6].view(6, 1), dd=both[:6]),
                 lambda: ops.selective_scan_bwd(x, x, x, a_log, bc, bc, saved, dd=both[:6], ddelta_bias=both[5:11]),
                 lambda: ops.layer_norm_bwd(x, x, None, stats, dweight=both[:6], dbias=both[:6])):
        with pytest.raises(ValueError, match='overlaps'):
            call()
    ops.layer_norm_bwd(x, x, None, stats, dweight=both[:6], dbias=both[6:12])


def test_launches_beyond_the_grid_are_refused():
    """Sizes whose launch would have 2^32 threads or more in one dimension: refused before anything is launched (pointers never read)."""
    from pb_sed_amd import _lib
    lib = _lib.lib()
    p = 1 << 20                                   # stands for any address
    big = 1 << 22
    strides = (ctypes.c_longlong * 16)()
    calls = [
        lambda: lib.pbsed_causal_conv_fwd(p, p, None, None, None, p, None, 1, 65535, big, 4, 65535 * big, big, 1, 0, 0, None),
        lambda: lib.pbsed_causal_conv_step(p, p, None, p, p, p, 65535, big, 4, big, 1, 0, None),
        lambda: lib.pbsed_causal_conv_step(p, p, None, p, p, p, 1, 2 * big, 4, 2 * big, 1, 0, None),
        lambda: lib.pbsed_selective_scan_fwd(p, p, p, p, p, None, None, None, None, None, p, None, None, None, 0, strides, 1, 1, big, 16, 1, 0, 0, None),
        lambda: lib.pbsed_layer_norm_fwd(p, None, None, p, None, 1, (1 << 24) + 1, (1 << 24) + 1, 1e-5, 0, None),
    ]
    for i, call in enumerate(calls):
        assert call() < 0, i
        assert lib.pbsed_last_error()


def test_cpu_tensors_are_refused():
    from pb_sed_amd import ops
    x = torch.zeros(4, 2, 6)
    for call in (lambda: ops.causal_conv_fwd(x, torch.zeros(6, 2)), lambda: ops.layer_norm_fwd(x), lambda: ops.dropout(x, .1, torch.zeros(2, dtype=torch.int64)),
                 lambda: ops.selective_scan_fwd(x, x, torch.zeros(6, 4), x[..., :4], x[..., :4])):
        with pytest.raises(RuntimeError, match='no CPU fallback'):
            call()


@pytest.mark.parametrize('entry', ['pbsed_causal_conv_fwd', 'pbsed_selective_scan_fwd', 'pbsed_selective_scan_bwd', 'pbsed_selective_scan_step',
                                   'pbsed_layer_norm_fwd', 'pbsed_layer_norm_bwd', 'pbsed_dropout', 'pbsed_causal_conv_step', 'pbsed_causal_conv_bwd'])
def test_entry_points_refuse_null_pointers_and_sizes(entry):
    """The C-ABI by itself: every pointer NULL, sizes of one and of nonsense - an error code and a message, no launch."""
    from pb_sed_amd import _lib
    lib = _lib.lib()
    for value in (1, 0, -5, 3):
        args = [None if t is ctypes.c_void_p else (ctypes.c_longlong * 16)() if hasattr(t, '_type_') and not isinstance(t._type_, str)
                else float(value) if t in (ctypes.c_double, ctypes.c_float) else value for t in _lib.SIGNATURES[entry]]
        assert getattr(lib, entry)(*args) < 0, value
        assert lib.pbsed_last_error()


# ------------------------------------------------------------------------------------------------ together
def layer(ops, x, p, rng, seq_len, reverse):
    """A state-space layer's operators one after the other (the projections between them are plain products): norm -> causal convolution
    -> scan with gate -> dropout and residual.  Returns the output and what the backward pass needs."""
    h, stats = ops.layer_norm_fwd(x, p['nw'], p['nb'], save=True)
    c, _ = ops.causal_conv_fwd(h, p['cw'], p['cb'], seq_len=seq_len, reverse=reverse)
    n = p['a_log'].shape[1]
    y, _, saved = ops.selective_scan_fwd(c, c, p['a_log'], c[..., :n], c[..., n:2 * n], d=p['d'], z=h, delta_bias=p['db'], seq_len=seq_len, reverse=reverse, save=True)
    return ops.dropout(y, .25, rng, site=2, residual=x), (h, stats, c, saved)


def layer_backward(ops, dout, x, p, rng, seq_len, reverse, kept, grads):
    h, stats, c, saved = kept
    n = p['a_log'].shape[1]
    dy = ops.dropout(dout, .25, rng, site=2)
    du, ddelta, db, dc, dz, _ = ops.selective_scan_bwd(dy, c, c, p['a_log'], c[..., :n], c[..., n:2 * n], saved, d=p['d'], z=h, delta_bias=p['db'],
                                                       seq_len=seq_len, reverse=reverse, da_log=grads['a_log'], dd=grads['d'], ddelta_bias=grads['db'])
    g = du + ddelta
    g[..., :n] += db
    g[..., n:2 * n] += dc
    dh, _ = ops.causal_conv_bwd(g, h, p['cw'], p['cb'], dweight=grads['cw'], dbias=grads['cb'], seq_len=seq_len, reverse=reverse)
    return dout + ops.layer_norm_bwd(dh + dz, x, p['nw'], stats, dweight=grads['nw'], dbias=grads['nb'])


def layer_parameters(g, d, n, dev):
    return {k: v.float().to(dev) for k, v in dict(nw=1 + normal(g, d, scale=.1), nb=normal(g, d, scale=.1), cw=normal(g, d, 4, scale=.5), cb=normal(g, d, scale=.1),
                                                  a_log=normal(g, d, n, scale=.3), d=normal(g, d), db=normal(g, d, scale=.3) - 1).items()}


@pytest.mark.parametrize('reverse', [False, True])
def test_layer_of_the_operators_against_autograd(dev, reverse):
    """The operators together, forward and backward, against the same layer written with float64 torch operations and its autograd
    gradients.  Bound: the layer's output is a chain of four operators, each within 2e-5 of its majorant for these sizes (100 u and a
    little); inputs of order one and a condition of a few per operator leave 1e-4 of the largest value."""
    from pb_sed_amd import ops
    t, b, d, n = 21, 2, 24, 8
    g = torch.Generator().manual_seed(12)
    p = layer_parameters(g, d, n, dev)
    x, dout = normal(g, t, b, d).float(), normal(g, t, b, d).float()
    seq_len = [21, 9]
    for i, m in enumerate(seq_len):
        dout[m:, i] = 0
    rng = torch.tensor([5, 6]).to(dev)
    grads = {k: torch.zeros_like(v) for k, v in p.items()}
    xd, ld = x.to(dev), lens(seq_len, dev)
    out, kept = layer(ops, xd, p, rng, ld, reverse)
    dx = layer_backward(ops, dout.to(dev), xd, p, rng, ld, reverse, kept, grads)

    q = {k: v.double().cpu().requires_grad_() for k, v in p.items()}
    x64 = x.double().requires_grad_()
    h = torch.nn.functional.layer_norm(x64, (d,), q['nw'], q['nb'], 1e-5)
    keep = torch.from_numpy(ref.philox_words(5, 6, 2, t * b * d) >= np.uint64(2 ** 30)).view(t, b, d)
    rows = []
    for i, m in enumerate(seq_len):
        hi = h[:m, i].flip(0) if reverse else h[:m, i]
        long = torch.cat([torch.zeros(3, d, dtype=torch.float64), hi])
        c = torch.nn.functional.silu(sum(long[j:j + m] * q['cw'][:, j] for j in range(4)) + q['cb'])
        s, ys = torch.zeros(d, n, dtype=torch.float64), []
        st = torch.nn.functional.softplus(c + q['db'])
        for f in range(m):
            s = torch.exp(-st[f][:, None] * q['a_log'].exp()) * s + (st[f] * c[f])[:, None] * c[f, :n][None]
            ys.append((s * c[f, n:2 * n]).sum(-1) + q['d'] * c[f])
        y = torch.stack(ys) * torch.nn.functional.silu(hi)
        y = y.flip(0) if reverse else y
        rows.append(torch.cat([y, torch.zeros(t - m, d, dtype=torch.float64)]))
    want = x64 + torch.where(keep, torch.stack(rows, 1) / .75, 0.)
    (want * dout.double()).sum().backward()

    def near(got, ref_, what):
        err = float((got.cpu().double() - ref_).abs().max() / ref_.abs().max())
        assert err < 1e-4, (what, err)
    near(out, want.detach(), 'out')
    near(dx, x64.grad, 'dx')
    for k in p:
        near(grads[k], q[k].grad, k)


# ------------------------------------------------------------------------------------------------ on the GPU only
@pytest.mark.gpu
def test_captured_layer_replays_with_new_masks_and_inputs():
    """Forward and backward of the layer captured into a graph: every replay equals the eager calls on the same inputs and mask, with eager
    work of the program between the replays; the step of the generator advances on the device."""
    from pb_sed_amd import ops
    dev = 'cuda:0'
    g = torch.Generator().manual_seed(4)
    t, b, d, n = 300, 2, 64, 16
    p = layer_parameters(g, d, n, dev)
    x, dout = normal(g, t, b, d).float().to(dev), normal(g, t, b, d).float().to(dev)
    seq_len, rng = lens([300, 190], dev), torch.tensor([9, 0]).to(dev)
    grads = {k: torch.zeros_like(v) for k, v in p.items()}

    def work(x, rng, grads):
        for v in grads.values():
            v.zero_()
        out, kept = layer(ops, x, p, rng, seq_len, True)
        return out, layer_backward(ops, dout, x, p, rng, seq_len, True, kept, grads)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(x, rng, grads)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, dx = work(x, rng, grads)
        rng[1] += 1
    for i in range(4):
        x.copy_(normal(torch.Generator().manual_seed(i), t, b, d))
        rng[1] = i
        own = {k: torch.zeros_like(v) for k, v in p.items()}
        want, wdx = work(x, rng.clone(), own)
        graph.replay()
        torch.cuda.synchronize()
        assert int(rng[1]) == i + 1
        assert torch.equal(out, want) and torch.equal(dx, wdx)
        assert all(torch.equal(grads[k], own[k]) for k in p)


@pytest.mark.gpu
def test_captured_frames_move_the_states_on():
    """The one-frame forms captured into a graph, states in place: replays on new inputs equal the eager calls, with eager work between."""
    from pb_sed_amd import ops
    dev = 'cuda:0'
    g = torch.Generator().manual_seed(5)
    b, d, n = 5, 70, 12
    p = layer_parameters(g, d, n, dev)
    x, bc = normal(g, b, d).float().to(dev), normal(g, b, 2 * n).float().to(dev)

    def frame(conv_state, state):
        u = ops.causal_conv_step(x, p['cw'], p['cb'], conv_state)
        return ops.selective_scan_step(u, x, p['a_log'], bc[:, :n], bc[:, n:], state, d=p['d'], z=x, delta_bias=p['db'])
    states = [torch.zeros(b, 3, d, device=dev), torch.zeros(b, d, n, device=dev)]
    own = [v.clone() for v in states]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        frame(*[v.clone() for v in states])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = frame(*states)
    for i in range(5):
        x.copy_(normal(torch.Generator().manual_seed(10 + i), b, d))
        want = frame(*own)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and all(torch.equal(u, v) for u, v in zip(states, own)), i
    assert float(states[1].abs().max()) > 0


@pytest.mark.gpu
def test_two_streams_and_repeated_calls_agree():
    """Calls on two streams at once (workspaces are per call) and repeated calls give the same bits."""
    from pb_sed_amd import ops
    dev = 'cuda:0'
    g = torch.Generator().manual_seed(8)
    p = layer_parameters(g, 128, 16, dev)
    xs = [normal(g, 400, 3, 128).float().to(dev) for _ in range(2)]
    dout, rng = normal(g, 400, 3, 128).float().to(dev), torch.tensor([1, 2]).to(dev)

    def work(x):
        grads = {k: torch.zeros_like(v) for k, v in p.items()}
        out, kept = layer(ops, x, p, rng, None, False)
        return [out, layer_backward(ops, dout, x, p, rng, None, False, kept, grads), *grads.values()]
    want = [work(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(work(x))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Tensors of more than 2^32 bytes and 2^31 elements: the last rows and frames equal the same rows and frames handled by themselves."""
    from pb_sed_amd import ops
    dev = 'cuda:0'
    rows, c = (1 << 21) + 3, 1025                                        # 2.15e9 elements of two bytes
    x = torch.empty(rows, c, dtype=BF16, device=dev)
    x[-40:] = normal(torch.Generator().manual_seed(0), 40, c)
    x[:40] = x[-40:]
    rng = torch.tensor([3, 4], device=dev)
    y = ops.dropout(x, .5, rng)
    first = (rows - 40) * c
    words = torch.tensor([int(w) for w in ref.philox_words_at(3, 4, 0, first, 64)], device=dev)
    assert torch.equal(y[-40:].reshape(-1)[:64] != 0, (words >= 1 << 31) & (x[-40:].reshape(-1)[:64] != 0))
    assert not torch.equal(y[-40:], y[:40])
    del y
    n, stats = ops.layer_norm_fwd(x, save=True)
    assert torch.equal(n[-40:], n[:40]) and torch.equal(n[-40:], ops.layer_norm_fwd(x[-40:].clone())[0])
    del n
    dx = ops.layer_norm_bwd(x, x, None, stats)
    assert torch.equal(dx[-40:], ops.layer_norm_bwd(x[-40:].clone(), x[-40:].clone(), None, stats[-40:].clone()))
    del x, dx, stats
    t, d = (1 << 22) + 70, 520                                           # [T, 1, D] half: 2.2e9 elements
    u = torch.zeros(t, 1, d, dtype=F16, device=dev)
    u[-200:] = normal(torch.Generator().manual_seed(1), 200, 1, d)
    w = normal(torch.Generator().manual_seed(2), d, 4).float().to(dev)
    y, last = ops.causal_conv_fwd(u, w, want_state=True)
    tail, tail_last = ops.causal_conv_fwd(u[-200:].clone(), w, want_state=True)
    assert torch.equal(y[-200:], tail) and torch.equal(last, tail_last) and (y[-300:-200] == 0).all()
    del y
    bc = torch.zeros(t, 1, 4, dtype=F16, device=dev)
    bc[-200:] = normal(torch.Generator().manual_seed(3), 200, 1, 4)
    a_log = torch.zeros(d, 4, device=dev)
    y, state, _ = ops.selective_scan_fwd(u, u, a_log, bc, bc, want_state=True)
    tail, tail_state, _ = ops.selective_scan_fwd(u[-200:].clone(), u[-200:].clone(), a_log, bc[-200:].clone(), bc[-200:].clone(), want_state=True)
    # the states start from zero in both; the long one meets it after another cut into runs
    assert torch.allclose(state, tail_state, rtol=1e-5, atol=1e-6) and torch.allclose(y[-200:].float(), tail.float(), rtol=2e-3, atol=1e-3)
    assert (y[:-200] == 0).all()
