"""Cases of the sequence operators that take a path of their own - element types, runs, several clips or channel blocks per sum, several turns of
a block - against the float64 restatements of tests/sequence_ref.py, on the emulated device (eight CUs) and on the GPU (256)."""
import pytest
import torch

from tests import sequence_ref as ref
from tests import test_sequence_ops as small
from tests.sequence_ref import check
from tests.test_sequence_ops import BF16, F16, F32, dev, emulated_library, normal, rounded, scan_inputs      # noqa: F401

name = lambda c: '-'.join(str(v) for v in c).replace(' ', '')        # noqa: E731

# t, b, d, n, seq_len, reverse, everything optional given, state, softplus, dtype
SCAN = [
    (260, 1, 4, 64, None, True, True, True, True, BF16),             # runs of four states per lane
    (260, 1, 5, 33, [200], False, True, True, True, F16),            # ... with states that do not exist; the last runs hold nothing
    (300, 2, 9, 20, [300, 171], False, False, False, True, BF16),    # runs of 16 lanes, nothing optional, no state
    (190, 1, 33, 12, None, True, True, False, True, F16),            # runs without a state in front
    (2304, 1, 2, 40, None, False, True, True, True, F32),            # more runs than the main launch folds
    (1000, 1, 3, 16, [989], False, True, True, True, BF16),
    (300, 1, 6, 12, [280], True, False, True, False, BF16),          # steps of either sign, in runs
    (300, 1, 4, 31, None, False, False, False, False, F32),
    (2, 520, 3, 4, None, False, True, True, True, F32),              # more rows of partial sums than a group of rows of the sums' launch
    (18, 2, 300, 16, [18, 5], False, True, True, True, F32),         # ten channel blocks
    (17, 1, 520, 7, None, True, True, False, True, BF16),            # nine of 64 channels
]


@pytest.mark.parametrize('case', SCAN, ids=name)
def test_selective_scan(dev, case):                                   # noqa: F811
    small.test_selective_scan_forward_and_gradients(dev, case, case[1] != 520)


# t, b, d, k, seq_len, reverse, state, silu, bias, dtype
CONV = [
    (1, 2100, 3, 4, None, False, True, True, True, F32),             # more rows of partial sums than a group of rows
    (300, 1, 7, 6, [290], True, True, True, True, BF16),
    (130, 2, 5, 7, [130, 3], False, True, True, True, F16),
]


@pytest.mark.parametrize('case', CONV, ids=name)
def test_causal_conv(dev, case):                                      # noqa: F811
    small.test_causal_conv_forward_and_gradients(dev, case, True)


@pytest.mark.parametrize('lead,c', small.NORM, ids=str)
@pytest.mark.parametrize('strided,affine', [(False, True), (True, False)])
def test_layer_norm_in_half_precision(dev, lead, c, strided, affine):     # noqa: F811
    small.test_layer_norm_forward_and_gradients(dev, lead, c, F16, strided, affine)


@pytest.mark.parametrize('rows,c', [(1500, 13), (600, 100), (150, 1023), (120, 1500), (40, 4100), (40, 8200)])
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_layer_norm_of_many_rows(dev, rows, c, dtype):                # noqa: F811
    """Blocks that walk several rows, with the weights' gradients."""
    from pb_sed_amd import ops
    if dev != 'cpu':
        rows *= 30
    g = torch.Generator().manual_seed(c)
    x, x64 = rounded(normal(g, rows, c) + normal(g, rows, 1), dtype)
    dy, dy64 = rounded(normal(g, rows, c), dtype)
    w, w64 = rounded(normal(g, c), F32)
    b, b64 = rounded(normal(g, c), F32)
    want = ref.layer_norm(x64, w64, b64, 1e-3, dy64)
    xd, gd, wd = x.to(dev), dy.to(dev), w.to(dev)
    y, stats = ops.layer_norm_fwd(xd, wd, b.to(dev), eps=1e-3, save=True)
    dw, db = torch.zeros(c, device=dev), torch.zeros(c, device=dev)
    dx = ops.layer_norm_bwd(gd, xd, wd, stats, dweight=dw, dbias=db)
    sums = 33 + 9                                                     # a lane's values one after the other, then the lanes' tree
    check(y, want['y'], want['major']['y'], 2 * sums + 8, 'y')
    check(dx, want['dx'], want['major']['dx'], 4 * sums + 20, 'dx')
    rows_ = min(rows, 256) + 16                                       # at most 256 turns in float, rows side by side; then double
    check(dw, want['dw'], want['major']['dw'], 2 * sums + 8 + rows_, 'dweight')
    check(db, want['db'], want['major']['db'], rows_ + 8, 'dbias')


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('k', [2, 4, 7])
def test_causal_conv_single_frames(dev, dtype, k):                    # noqa: F811
    """One frame of several streams against the restatement; in place and into another buffer."""
    from pb_sed_amd import ops
    g = torch.Generator().manual_seed(k)
    b, d = 7, 133
    x, x64 = rounded(normal(g, 1, b, d), dtype)
    state, state64 = rounded(normal(g, b, k - 1, d), dtype)
    w, w64 = rounded(normal(g, d, k, scale=k ** -.5), F32)
    bias, bias64 = rounded(normal(g, d), F32)
    xd, wd, bd, sd = small.slot(x[0], dev), w.to(dev), bias.to(dev), state.to(dev)
    for silu in (True, False):
        want = ref.conv(x64, w64, bias64, silu=silu, state=state64)
        other = torch.empty_like(sd)
        y = ops.causal_conv_step(xd, wd, bd, sd, silu=silu, state_out=other)
        check(y, want['y'][0], want['major']['y'][0], k + 10, 'y')
        assert torch.equal(other.cpu().double(), want['state_out']) and torch.equal(sd.cpu(), state)
    y2 = ops.causal_conv_step(xd, wd, bd, sd, silu=False)
    assert torch.equal(y2, y) and torch.equal(sd, other)


@pytest.mark.parametrize('n', [4, 16, 23])
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_selective_scan_single_frames_of_many_streams(dev, n, dtype):     # noqa: F811
    """Blocks that keep the rates of their channels over several clips and fetch the next clip early; in place as well."""
    from pb_sed_amd import ops
    g = torch.Generator().manual_seed(n)
    b, d = (150, 70) if dev == 'cpu' else (390, 1030)
    v, v64 = scan_inputs(g, 1, b, d, n, dtype, True, True)
    step = torch.nn.functional.softplus(v64['delta'][0] + v64['delta_bias'], threshold=100)
    rate = -torch.exp(v64['a_log'])
    decay = torch.exp(step[..., None] * rate)
    drive = (step * v64['u'][0])[..., None] * v64['b'][0][:, None]
    h = decay * v64['state'] + drive
    pre = (h * v64['c'][0][:, None]).sum(-1) + v64['d'] * v64['u'][0]
    gate = v64['z'][0] * torch.sigmoid(v64['z'][0])
    # the majorants of sequence_ref.scan for one frame
    raw_major = v64['delta'][0].abs() + v64['delta_bias'].abs()
    step_major = step + torch.sigmoid(v64['delta'][0] + v64['delta_bias']) * raw_major
    h_major = decay * v64['state'].abs() * (2 + step_major[..., None] * rate.abs()) + (step_major * v64['u'][0].abs())[..., None] * v64['b'][0].abs()[:, None]
    pre_major = (h_major * v64['c'][0].abs()[:, None]).sum(-1) + (v64['d'] * v64['u'][0]).abs()
    x = {key: t[0].to(dev) if key in ('u', 'delta', 'b', 'c', 'z') else t.to(dev) for key, t in v.items()}
    args, kw = [x[key] for key in ('u', 'delta', 'a_log', 'b', 'c')], dict(d=x['d'], z=x['z'], delta_bias=x['delta_bias'])
    other = torch.empty_like(x['state'])
    y = ops.selective_scan_step(*args, x['state'], state_out=other, **kw)
    check(y, pre * gate, pre_major * gate.abs() + (pre * v64['z'][0]).abs() * .3, 30 + n, 'y')
    check(other, h, h_major, 20, 'state')
    assert torch.equal(x['state'].cpu(), v['state'])
    again = ops.selective_scan_step(*args, x['state'], **kw)
    assert torch.equal(again, y) and torch.equal(x['state'], other)
