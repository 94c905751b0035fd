"""The sequence operators of pb_sed_amd.ops at the edges of their ranges, against the float64 restatements of tests/sequence_ref.py: on the
GPU and on the emulated device (whose eight CUs cut small cases into runs as well)."""
import numpy as np
import pytest
import torch

from tests import sequence_ref as ref
from tests.sequence_ref import check
from tests.test_sequence_ops import BF16, F16, F32, dev, emulated_library, lens, normal, rounded, scan_inputs, slot      # noqa: F401


def up(v, dev):                                                       # noqa: F811
    return {k: x.to(dev) for k, x in v.items()}


def scan_forward(ops, v, n=None, **kw):
    """(y, state behind the frames) of inputs ``v`` (frames from n[0] to n[1])."""
    cut = {k: v[k][slice(*n)] if n else v[k] for k in ('u', 'delta', 'b', 'c')}
    return ops.selective_scan_fwd(cut['u'], cut['delta'], v['a_log'], cut['b'], cut['c'], want_state=True, **kw)[:2]


# ------------------------------------------------------------------------------------------------ scans that grow
# softplus=False takes steps below zero, whose factors exp(D A) are above one: over a run of 48 frames (what T >= 128 frames of few clips
# and channels are cut into) their product leaves float32 long before a result does.
def growing(t, d, n, step=-3.):
    g = torch.Generator().manual_seed(t + n)
    v = dict(u=torch.zeros(t, 1, d), delta=torch.full((t, 1, d), step), b=normal(g, t, 1, n).float(), c=normal(g, t, 1, n).float(), a_log=torch.zeros(d, n),
             dy=torch.zeros(t, 1, d))
    return v


@pytest.mark.parametrize('n', [4, 16, 20, 64])
@pytest.mark.parametrize('reverse', [False, True])
def test_growing_scans_cut_into_runs_stay_zero_until_they_are_driven(dev, n, reverse):      # noqa: F811
    """390 silent frames whose factors multiply up to exp(1170), then ten of input: the state is 0 until then.  Backward: only the first
    ten frames have a gradient, and the adjoint is 0 behind them."""
    from pb_sed_amd import ops
    t, d = 400, 5
    v = growing(t, d, n)
    last = slice(0, 10) if reverse else slice(390, 400)               # the last ten, the first ten frames in scan order
    first = slice(390, 400) if reverse else slice(0, 10)
    v['u'][last] = 1.
    v['dy'][first] = 1.
    x = up(v, dev)
    want = ref.scan(*(v[k].double() for k in ('u', 'delta', 'a_log', 'b', 'c')), softplus=False, reverse=reverse, dy=v['dy'].double())
    args = [x[k] for k in ('u', 'delta', 'a_log', 'b', 'c')]
    y, state, saved = ops.selective_scan_fwd(*args, softplus=False, reverse=reverse, want_state=True, save=True)
    k = 30 + 64                                                       # (as in test_sequence_ops: 30 per frame, a sum of D over a run)
    check(y, want['y'], want['major']['y'], k, 'y')
    check(state, want['state_out'], want['major']['state_out'], k, 'state_out')
    silent = torch.ones(t, dtype=torch.bool)
    silent[last] = False
    assert (y.cpu()[silent] == 0).all()
    da, dd, db = torch.zeros(d, n, device=dev), torch.zeros(d, device=dev), torch.zeros(d, device=dev)
    got = ops.selective_scan_bwd(x['dy'], *args, saved, softplus=False, reverse=reverse, da_log=da, dd=dd, ddelta_bias=db, want_dstate=True)
    k = 2 * k + 20 + 16 + t // 16
    for key, value in (*zip(('du', 'ddelta', 'db', 'dc'), got), ('dstate', got[5]), ('da_log', da), ('dd', dd), ('ddelta_bias', db)):
        check(value, want[key], want['major'][key], k, key)


def test_growing_scans_do_not_depend_on_the_cut(dev):                 # noqa: F811
    """The cut call, the same frames in uncut pieces and frame by frame: a state that is cancelled at the border of two runs, and one so
    small that only the product of a run's factors with it is within float32."""
    from pb_sed_amd import ops
    t, d, n = 144, 3, 4
    v = growing(t, d, n, step=0.)
    v['a_log'].fill_(float(np.log(np.log(2.))))                       # factor 2^-D
    v['b'].fill_(1.)
    start = torch.zeros(1, d, n)
    # channel 0: the state 1 meets -8 in frame 48 and would grow 8-fold in the 47 frames behind it, as would the input alone: 2^141
    start[:, 0] = 1.
    v['delta'][48:96, :, 0] = -3.
    v['u'][48, :, 0] = 8 / 3
    # channel 1: 2^-140 grows by 2^200 in frames 48 .. 95 and is held; channel 2: shrinks by 2^200, then grows by it
    start[:, 1] = 2. ** -120
    v['delta'][48:96, :, 1] = -200 / 48
    start[:, 2] = 2. ** 100
    v['delta'][:48, :, 2] = 200 / 48
    v['delta'][48:96, :, 2] = -200 / 48
    x, h0 = up(v, dev), start.to(dev)
    want = ref.scan(*(v[k].double() for k in ('u', 'delta', 'a_log', 'b', 'c')), softplus=False, state=start.double())
    y, state = scan_forward(ops, x, softplus=False, state=h0)
    check(y, want['y'], want['major']['y'], 94, 'y')
    check(state, want['state_out'], want['major']['state_out'], 94, 'state_out')
    pieces, h = [], h0
    for a in range(0, t, 36):                                         # 36 frames are not cut
        p, h = scan_forward(ops, x, (a, a + 36), softplus=False, state=h)
        pieces.append(p)
    check(torch.cat(pieces), want['y'], want['major']['y'], 94, 'y in pieces')
    h = h0.clone()
    for f in range(t):
        one = ops.selective_scan_step(x['u'][f], x['delta'][f], x['a_log'], x['b'][f], x['c'][f], h, softplus=False)
        check(one, want['y'][f], want['major']['y'][f], 94, f'frame {f}')
    check(h, want['state_out'], want['major']['state_out'], 94, 'state, frame by frame')


def test_growing_scans_that_leave_float32_stay_outside(dev):          # noqa: F811
    """Driven from the first frame: finite up to float32's range as in the formula, and not finite in any run behind that."""
    from pb_sed_amd import ops
    t, d, n = 400, 5, 4
    v = growing(t, d, n)
    v['u'][:20] = 1.
    v['b'].abs_(), v['c'].abs_().add_(.5)
    want = ref.scan(*(v[k].double() for k in ('u', 'delta', 'a_log', 'b', 'c')), softplus=False)
    y, state = scan_forward(ops, up(v, dev), softplus=False)
    inside = want['y'].abs() < 1e37                                   # (the states too: c >= 0.5)
    assert inside.any() and not inside.all() and not torch.isfinite(y.cpu()[want['y'].abs() > 1e39]).any()
    check(y.cpu()[inside], want['y'][inside], want['major']['y'][inside], 94, 'y')
    assert not torch.isfinite(state).any()


# ------------------------------------------------------------------------------------------------ infinities beside padding
# States are padded to 8, 16, 32 or 64 and channels to a block; an infinity that the formula keeps must not meet their zeros.
def same(got, want, what):
    """NaN, infinities and their signs as in the formula.  The rest: at most 237 roundings (2 (30 + 64) of a state and an adjoint, 49 of the
    sums) against majorants that exceed these positive sums at most 20-fold (1 + the sum of D rate <= 19): 3e-4."""
    got = got.detach().cpu().double()
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(kind(got), kind(want)), (what, kind.__name__, kind(got).nonzero()[:5].tolist(), kind(want).nonzero()[:5].tolist())
    fin = torch.isfinite(want)
    err = (got[fin] - want[fin]).abs()
    assert (err <= 3e-4 * want[fin].abs().clamp(min=1e-30)).all(), (what, float((err / want[fin].abs().clamp(min=1e-30)).max()))


# (160 frames: cut into runs)
@pytest.mark.parametrize('t,n', [(32, 1), (32, 3), (32, 8), (32, 12), (32, 16), (32, 19), (32, 20), (32, 33), (32, 62), (160, 5), (160, 12), (160, 33)])
@pytest.mark.parametrize('where', ['u', 'delta', 'b', 'c', 'dy'])
def test_infinities_do_not_meet_the_padding(dev, t, n, where):        # noqa: F811
    from pb_sed_amd import ops
    d = 33 if t == 32 else 5
    g = torch.Generator().manual_seed(n)
    v = dict(u=(t, 1, d), delta=(t, 1, d), b=(t, 1, n), c=(t, 1, n), dy=(t, 1, d), d=(d,), delta_bias=(d,))
    v = {k: .5 + torch.rand(*s, generator=g) for k, s in v.items()}
    v['delta_bias'] -= 1.5
    v['a_log'] = torch.full((d, n), -2.5)                             # D rate <= 0.13
    v[where][{'c': 12, 'dy': 12}.get(where, 7), 0, 0 if where in 'bc' else 2] = float('inf')
    want = ref.scan(*(v[k].double() for k in ('u', 'delta', 'a_log', 'b', 'c')), dy=v['dy'].double(), d=v['d'].double(), delta_bias=v['delta_bias'].double())
    x = up(v, dev)
    args, kw = [x[k] for k in ('u', 'delta', 'a_log', 'b', 'c')], dict(d=x['d'], delta_bias=x['delta_bias'])
    y, state, saved = ops.selective_scan_fwd(*args, want_state=True, save=True, **kw)
    same(y, want['y'], 'y')
    same(state, want['state_out'], 'state_out')
    da, dd, db = torch.zeros(d, n, device=dev), torch.zeros(d, device=dev), torch.zeros(d, device=dev)
    got = ops.selective_scan_bwd(x['dy'], *args, saved, da_log=da, dd=dd, ddelta_bias=db, want_dstate=True, **kw)
    for key, value in (*zip(('du', 'db', 'dc'), (got[0], *got[2:4])), ('dstate', got[5]), ('dd', dd)):
        same(value, want[key], key)
    for key, value in (('ddelta', got[1]), ('da_log', da), ('ddelta_bias', db)):         # (differences)
        assert torch.equal(torch.isfinite(value.cpu()), torch.isfinite(want[key])), key
    h = torch.zeros(1, d, n, device=dev)
    for f in range(20 if where in ('u', 'delta', 'b', 'c') else 0):
        one = ops.selective_scan_step(x['u'][f], x['delta'][f], x['a_log'], x['b'][f], x['c'][f], h, **kw)
        same(one, want['y'][f], f'frame {f}')


def test_infinities_without_the_skip_weight(dev):                     # noqa: F811
    """d=None: there is no term for it, and none whose 0 an infinite input or gradient could meet."""
    from pb_sed_amd import ops
    g = torch.Generator().manual_seed(1)
    t, d, n = 20, 5, 8
    u, delta, b, c, z, dy = (.5 + torch.rand(t, 1, k, generator=g) for k in (d, d, n, n, d, d))
    u[7, 0, 2], dy[12, 0, 3] = float('inf'), float('inf')
    a_log = torch.full((d, n), -2.5)
    u, delta, a_log, b, c, z, dy = (v.to(dev) for v in (u, delta, a_log, b, c, z, dy))
    y, _, saved = ops.selective_scan_fwd(u, delta, a_log, b, c, z=z, save=True)
    du, _, _, _, dz, _ = ops.selective_scan_bwd(dy, u, delta, a_log, b, c, saved, z=z)
    inf = torch.zeros(t, 1, d, dtype=torch.bool)
    inf[7:, 0, 2] = True                                              # the state is infinite from there on
    assert torch.equal(torch.isposinf(y.cpu()), inf) and torch.isfinite(y.cpu()[~inf]).all()
    inf[12, 0, 3] = True
    assert torch.equal(torch.isposinf(dz.cpu()), inf) and torch.isfinite(dz.cpu()[~inf]).all()
    inf.zero_()
    inf[:13, 0, 3] = True                                             # the adjoint is, up to there
    assert torch.equal(torch.isposinf(du.cpu()), inf) and torch.isfinite(du.cpu()[~inf]).all()
    h = torch.zeros(1, d, n, device=dev)
    for f in range(10):
        one = ops.selective_scan_step(u[f], delta[f], a_log, b[f], c[f], h, z=z[f])
        assert torch.equal(torch.isposinf(one.cpu()), torch.isposinf(y[f].cpu())) and not torch.isnan(one).any(), f


# ------------------------------------------------------------------------------------------------ memory that is read and written
def test_outputs_over_operands_are_refused(dev):                      # noqa: F811
    """What a launch writes must not be what it still reads, nor another output: refused before anything is launched."""
    from pb_sed_amd import ops
    t, b, d, k, n = 4, 2, 6, 4, 5
    f = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype, device=dev)     # noqa: E731
    over = lambda v, *s, off=0: v.flatten()[off:off + int(np.prod(s))].view(s)   # noqa: E731
    arena = f(600)
    x, w, bias, cs = f(t, b, d), f(d, k), f(d), f(b, k - 1, d)
    u, al, bc, h = f(t, b, d), f(d, n), f(t, b, n), f(b, d, n)
    saved = ops.selective_scan_fwd(u, u, al, bc, bc, save=True)[2]
    stats = ops.layer_norm_fwd(x, save=True)[1]
    conv_bwd = lambda **o: ops.causal_conv_bwd(o.pop('dy', x.clone()), o.pop('x', x), o.pop('w', w), o.pop('bias', bias), **o)        # noqa: E731
    scan_bwd = lambda **o: ops.selective_scan_bwd(**{**dict(dy=u, u=u, delta=u, a_log=al, b=bc, c=bc, saved=saved), **o})             # noqa: E731
    step = lambda **o: ops.selective_scan_step(**{**dict(u=u[0], delta=u[0], a_log=al, b=bc[0], c=bc[0], state=h), **o})              # noqa: E731
    norm_bwd = lambda **o: ops.layer_norm_bwd(x, o.pop('x', x), o.pop('w', bias), o.pop('stats', stats), **o)                         # noqa: E731
    state, near, head, frame = over(arena, b, k - 1, d), over(arena, b, d, off=30), over(arena, d, off=35), over(arena, t, b, d, off=3)
    big = over(arena, b, d, n)
    shared = over(saved, t, b, d)
    refused = [
        lambda: ops.causal_conv_step(near, w, bias, state), lambda: ops.causal_conv_step(near, w, bias, cs, state_out=state),
        lambda: ops.causal_conv_step(x[0], over(arena, d, k, off=20), bias, cs, state_out=state), lambda: ops.causal_conv_step(x[0], w, head, cs, state_out=state),
        lambda: ops.causal_conv_step(x[0], w, head, state),
        lambda: conv_bwd(w=over(arena, d, k), dx=frame), lambda: conv_bwd(bias=over(arena, d, off=50), dx=frame), lambda: conv_bwd(state=state, dx=frame),
        lambda: conv_bwd(dweight=over(arena, d, k), dx=frame), lambda: conv_bwd(dbias=over(arena, d, off=50), dx=frame),
        lambda: conv_bwd(dweight=w), lambda: conv_bwd(dbias=bias), lambda: conv_bwd(x=frame, dweight=over(arena, d, k)), lambda: conv_bwd(dy=frame, dbias=head),
        lambda: conv_bwd(state=state, dweight=over(arena, d, k)), lambda: conv_bwd(dstate_out=state, dweight=over(arena, d, k)),
        lambda: scan_bwd(z=u, dz=shared), lambda: scan_bwd(z=u, dz=frame, dstate_out=big), lambda: scan_bwd(z=u, dz=frame, da_log=over(arena, d, n)),
        lambda: scan_bwd(z=u, dz=frame, dd=head), lambda: scan_bwd(z=u, dz=frame, ddelta_bias=head), lambda: scan_bwd(z=u, dz=frame, a_log=over(arena, d, n)),
        lambda: scan_bwd(da_log=al), lambda: scan_bwd(dd=over(u, d)), lambda: scan_bwd(ddelta_bias=over(saved, d)), lambda: scan_bwd(d=head, dd=head),
        lambda: scan_bwd(da_log=over(bc, d, n)), lambda: scan_bwd(dstate_out=big, da_log=over(arena, d, n)),
        lambda: step(state=big, u=near), lambda: step(state_out=big, delta=near), lambda: step(state_out=big, b=over(arena, b, n, off=7)),
        lambda: step(state_out=big, c=over(arena, b, n, off=7)), lambda: step(state_out=big, z=near), lambda: step(state_out=big, a_log=over(arena, d, n, off=9)),
        lambda: step(state_out=big, d=head), lambda: step(state_out=big, delta_bias=head), lambda: step(state=big, a_log=over(arena, d, n, off=9)),
        lambda: norm_bwd(dweight=bias), lambda: norm_bwd(dbias=over(x, d)), lambda: norm_bwd(dbias=over(stats, d)),
    ]
    for i, call in enumerate(refused):
        with pytest.raises((ValueError, RuntimeError), match='overlaps'):
            call()
            raise AssertionError(f'call {i} was accepted')
    # neighbours in one buffer are no overlap
    ops.causal_conv_step(over(arena, b, d, off=36), w, over(arena, d, off=48), state)
    ops.causal_conv_bwd(x.clone(), x, w, bias, dweight=over(arena, d, k), dbias=over(arena, d, off=24), dx=over(arena, t, b, d, off=30))
    step(state=over(arena, b, d, n), u=over(arena, b, d, off=60), a_log=over(arena, d, n, off=72))
    wide = f(t, b, 2 * d)
    ops.causal_conv_bwd(wide[..., d:], x, w, bias, dx=wide[..., :d])
    scan_bwd(dy=wide[..., d:], z=u, dz=wide[..., :d])


def test_launches_beyond_the_grid_are_named():
    """Refused for their size (pointers, never read, would be refused as overlapping behind that): the message names the blocks or the
    limit.  The scan's last launch holds blocks for the parameters' sums and for dB, dC: together less than 2^32 threads."""
    import ctypes
    from pb_sed_amd import _lib
    lib = _lib.lib()
    p, big, strides = 1 << 20, 1 << 22, (ctypes.c_longlong * 16)()
    scan = lambda d, n, sums: lib.pbsed_selective_scan_bwd(p, p, p, p, p, p, None, None, None, None, p, None, p, p, p, p, None, None, p if sums else None, None, None,  # noqa: E731
                                                           p, 1 << 50, strides, 300, 1, d, n, 1, 0, 0, None)
    calls = [
        (lambda: lib.pbsed_causal_conv_fwd(p, p, None, None, None, p, None, 1, 65535, big, 4, 65535 * big, big, 1, 0, 0, None), 'blocks'),
        (lambda: lib.pbsed_causal_conv_step(p, p, None, p, p, p, 65535, big, 4, big, 1, 0, None), 'blocks'),
        (lambda: scan(8388600, 6, True), 'blocks'),            # 4194300 blocks of sums, at least 5 of dB and dC
        (lambda: scan(8388600, 6, False), 'overlaps'),
        (lambda: scan(8388400, 6, False), 'overlaps'),
        (lambda: scan(1 << 18, 254, True), 'N <= 64'),
    ]
    for i, (call, word) in enumerate(calls):
        assert call() < 0 and word in lib.pbsed_last_error().decode(), (i, lib.pbsed_last_error())


# ------------------------------------------------------------------------------------------------ sums over long axes
def test_sums_of_long_uncut_scans_keep_their_digits(dev):             # noqa: F811
    """Terms of one sign over many frames of a scan that is not cut into runs (clips and channels fill the device): the bound counts a tile's
    terms, the 32 tiles that are added in float and the groups of frames of a block - 16 + 32 + 16 + 4 roundings - not the frames."""
    from pb_sed_amd import ops
    t, b = (3500, 10) if dev == 'cpu' else (20000, 300)
    d, n = 2, 2
    # 4/3: every addition to a sum is off by a third of its last place, in one direction while the sum's exponent lasts
    u, dy, delta = torch.full((t, b, d), 4 / 3), torch.ones(t, b, d), torch.full((t, b, d), .7)
    bm, cm = torch.ones(t, b, n), torch.ones(t, b, n)
    a_log, skip = torch.zeros(d, n), torch.ones(d)
    x = [v.to(dev) for v in (u, delta, a_log, bm, cm)]
    _, _, saved = ops.selective_scan_fwd(*x, d=skip.to(dev), save=True)
    da, dd, db = torch.zeros(d, n, device=dev), torch.zeros(d, device=dev), torch.zeros(d, device=dev)
    ddelta = ops.selective_scan_bwd(dy.to(dev), *x, saved, d=skip.to(dev), da_log=da, dd=dd, ddelta_bias=db)[1]
    k = 16 + 32 + 16 + 4
    want = b * (dy[:, 0].double() * u[:, 0].double()).sum(0)
    check(dd, want, want, k, 'dd')
    terms = ddelta.double().cpu()
    check(db, terms.sum((0, 1)), terms.abs().sum((0, 1)), k, 'ddelta_bias')      # (the launch's own float terms)
    # da_log against the recurrence in float64: D, exp, h and r carry some 30 roundings of a frame each, for a factor of 0.27
    # and less per frame (1 / (1 - 0.27)): 2 x 42 more
    step = torch.nn.functional.softplus(delta[:, 0].double())[..., None]
    decay, drive = torch.exp(-step), step * (u[:, 0, :, None] * bm[:, 0, None]).double()
    h, past = torch.zeros(d, n, dtype=torch.float64), []
    for f in range(t):
        past.append(h)
        h = decay[f] * h + drive[f]
    r, want = torch.zeros(d, n, dtype=torch.float64), torch.zeros(d, n, dtype=torch.float64)
    for f in reversed(range(t)):
        r = r + dy[f, 0, :, None].double() * cm[f, 0, None].double()
        want -= r * decay[f] * past[f] * step[f]
        r = r * decay[f]
    check(da, b * want, b * want.abs(), k + 2 * 42, 'da_log')


@pytest.mark.parametrize('c,rows', [(9, 140_000), (300, 10_000), (9000, 2500)])      # more than 256 turns of eight CUs
def test_sums_of_many_rows_keep_their_digits(dev, c, rows):           # noqa: F811
    """Layer norm's weight gradients over rows whose terms have one sign: a block adds at most 256 turns in float."""
    from pb_sed_amd import ops
    if dev != 'cpu':
        rows = {9: 40_000_000, 300: 10_000_000, 9000: 500_000}[c]     # thousands of turns of 256 CUs
    row = normal(torch.Generator().manual_seed(c), 1, c).float()
    x = row.to(dev).expand(rows, c).contiguous()
    dy = torch.full((rows, c), 4 / 3, device=dev)                     # (as above)
    _, stats = ops.layer_norm_fwd(x, save=True)
    dw, db = torch.zeros(c, device=dev), torch.zeros(c, device=dev)
    ops.layer_norm_bwd(dy, x, None, stats, dweight=dw, dbias=db)
    want = rows * dy[0].double().cpu()
    k = 256 + 16 + 2                                                  # turns, rows of a block side by side, two conversions
    check(db, want, want, k, 'dbias')
    mean, rstd = stats[0].double().cpu()
    xh = (row[0].double() - mean) * rstd                              # (two roundings of a term: the difference and the product)
    check(dw, want * xh, (want * xh).abs(), k + 3, 'dweight')
