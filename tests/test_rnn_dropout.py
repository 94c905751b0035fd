"""Dropout between GRU layers (torch.nn.GRU's ``dropout``; the recurrent layers of pb_sed/models/weak_label/crnn.py:61-67): the engine's
recurrent forward and backward against float64 GRU cells with the generator's own masks; on the emulated device and on the GPU."""
import warnings

import numpy as np
import pytest
import torch

from tests.sequence_ref import philox_words


@pytest.fixture(scope='module')
def emulated_library(tmp_path_factory):
    from tests.emu import cpu_device
    return cpu_device.EmulatedLibrary(tmp_path_factory.mktemp('emu_rnn'))


@pytest.fixture(params=['emulated', pytest.param('cuda', marks=pytest.mark.gpu)])
def dev(request, monkeypatch):
    if request.param == 'cuda':
        yield 'cuda:0'
        return
    from tests.emu import cpu_device
    with cpu_device.emulated_device(monkeypatch, request.getfixturevalue('emulated_library')):
        yield 'cpu'


def cell_scan(x, w_ih, b_ih, w_hh, b_hh, order, t):
    """One clip through one GRU direction: x [T, In] -> [T, H], zeros where the clip has no frame."""
    hid = w_hh.shape[1]
    h = x.new_zeros(hid)
    out = [x.new_zeros(hid)] * t
    for f in order:
        gi, gh = w_ih @ x[f] + b_ih, w_hh @ h + b_hh
        r, z = torch.sigmoid(gi[:hid] + gh[:hid]), torch.sigmoid(gi[hid:2 * hid] + gh[hid:2 * hid])
        n = torch.tanh(gi[2 * hid:] + r * gh[2 * hid:])
        h = (1 - z) * n + z * h
        out[f] = h
    return torch.stack(out)


@pytest.mark.parametrize('kind', ['forward_and_reversed', 'bidirectional'])
def test_dropout_between_gru_layers(dev, kind, monkeypatch):
    """Outputs and every gradient of two- and three-layer stacks.  Bound: the recurrent path is compared at 1e-4 of the largest value
    (gradients 1e-3), as the GRU scans are elsewhere; dropout adds two roundings per layer."""
    from pb_sed_amd import engine, modules
    # heads left out: the recurrent part's outputs and the gradients that reach them are what is compared
    monkeypatch.setattr(engine, '_heads_forward', lambda ws, x_w, *a, x_tbc=None, **k: (list(x_tbc), [(None, None)] * len(ws)))
    monkeypatch.setattr(engine, 'stack_backward', lambda layers, c, g, *a, **k: g)
    torch.manual_seed(3)
    p, b, t, cin, hid = .3, 2, 5, 8, 64
    with warnings.catch_warnings():
        warnings.simplefilter('error')
        if kind == 'bidirectional':
            wrappers = [modules.build_rnn(cin, hid, 3, 4, 16, bidirectional=True, dropout=p)]
        else:
            wrappers = [modules.build_rnn(cin, hid, 2, 4, 16, reverse=r, dropout=p) for r in (False, True)]
    for w in wrappers:
        w.to(dev)
    layers = wrappers[0].num_layers
    h = torch.randn(b, cin, t)
    seq = np.array([5, 3])
    seq_dev = torch.tensor(seq, dtype=torch.int32).to(dev)
    outs, ctx = engine.rnn_forward(wrappers, h.to(dev), seq_dev, seq, True)
    # (the state advanced once per wrapper; the pass drew from the step before)
    states = [tuple(int(v) for v in w.dropout_rng.tolist()) for w in wrappers]
    assert all(step == 1 for _, step in states)
    width = hid * (2 if kind == 'bidirectional' else 1)
    dlogits = [torch.randn(b, width, t) for _ in wrappers]
    for d in dlogits:
        d[1, :, 3:] = 0
    dh = engine.rnn_backward(wrappers, ctx, [d.to(dev) for d in dlogits], seq_dev, seq)

    h64 = h.double().requires_grad_()
    loss, params = 0., []
    for wi, w in enumerate(wrappers):
        own = {k: v.detach().double().cpu().requires_grad_() for k, v in w.rnn.named_parameters()}
        params.append(own)
        x = h64.permute(2, 0, 1)                                        # [T, B, C]
        dirs = 2 if w.bidirectional else 1
        for l in range(layers):
            parts = []
            for d in range(dirs):
                suffix = f'_l{l}' + ('_reverse' if d else '')
                rev = bool(w.reverse) ^ bool(d)
                one = torch.stack([cell_scan(x[:, i], *(own[k + suffix] for k in ('weight_ih', 'bias_ih', 'weight_hh', 'bias_hh')),
                                             [*range(n)][::-1] if rev else range(n), t) for i, n in enumerate(seq)], 1)
                if l + 1 < layers:
                    chain = wi * dirs + d
                    words = philox_words(states[wi][0], 0, 8 * l + chain, one.numel())
                    one = torch.where(torch.from_numpy(words >= np.uint64(int(p * 2 ** 32))).view(one.shape), one / (1 - p), 0.)
                parts.append(one)
            x = torch.cat(parts, 2)
        got = outs[wi].cpu().double()
        assert float((got - x.detach()).abs().max()) < 1e-4, wi
        loss = loss + (x * dlogits[wi].double().permute(2, 0, 1)).sum()
    loss.backward()

    def near(got, want, what):
        err = float((got.cpu().double() - want).abs().max() / want.abs().max())
        assert err < 1e-3, (what, err)
    near(dh, h64.grad, 'dh')
    for w, own in zip(wrappers, params):
        for k, v in w.rnn.named_parameters():
            near(v.grad, own[k].grad, k)
    # inference draws nothing, and a second training pass other masks
    again, _ = engine.rnn_forward(wrappers, h.to(dev), seq_dev, seq, True)
    assert not torch.equal(again[0], outs[0])
    plain, _ = engine.rnn_forward(wrappers, h.to(dev), seq_dev, seq, False)
    for w in wrappers:
        w.rnn.dropout = 0.
    bare, _ = engine.rnn_forward(wrappers, h.to(dev), seq_dev, seq, False)
    assert all(torch.equal(a, c) for a, c in zip(plain, bare))
    assert all(int(w.dropout_rng[1]) == 2 for w in wrappers)


def test_gru_dropout_configuration():
    """Constructor range, one-layer networks, and the model factories."""
    from pb_sed_amd import modules
    from pb_sed_amd.models import strong_label, weak_label
    with pytest.raises(NotImplementedError, match='dropout'):
        modules.GRU(torch.nn.GRU(8, 64, 2, batch_first=True, dropout=1.))
    with warnings.catch_warnings():
        warnings.simplefilter('ignore')                                 # torch: dropout has no effect in one layer
        assert modules.GRU(torch.nn.GRU(8, 64, 1, batch_first=True, dropout=.5)).dropout == 0.
    model = weak_label.CRNN.build(rnn_dropout=.2)
    assert model.rnn_fwd.dropout == model.rnn_bwd.dropout == .2 and weak_label.CRNN.build().rnn_fwd.dropout == 0.
    assert strong_label.CRNN.build(rnn_dropout=.1).rnn.dropout == .1
    assert model.state_dict().keys() == weak_label.CRNN.build().state_dict().keys()


@pytest.mark.gpu
def test_training_step_with_gru_dropout_on_the_gpu():
    """A whole training step of both models with dropout between the GRU layers: finite gradients everywhere, other masks every step, and
    evaluation as without it."""
    from pb_sed_amd.models import strong_label, weak_label
    net = dict(out_channels_2d=[16, 16, 32], pool_sizes_2d=[1, (2, 1), (2, 1)], kernel_size_2d=3, out_channels_1d=[64, 64], kernel_size_1d=[1, 3])
    wav, seq = torch.randn(3, 16000).cuda(), [50, 40, 33]
    weak = (torch.rand(3, 10) < .4).float().cuda()
    for cls, more in ((weak_label.CRNN, dict(boundary_targets=torch.rand(3, 10, 50).round().cuda())),
                      (strong_label.CRNN, dict(strong_targets=torch.rand(3, 10, 50).round().cuda(), tag_condition=weak))):
        torch.manual_seed(0)
        model = cls.build(num_events=10, hidden_size=64, num_layers=2, net=net, rnn_dropout=.25).cuda()
        inputs = lambda: {'audio_data': wav, 'seq_len': list(seq), 'weak_targets': weak, **more}      # noqa: E731
        losses = []
        model.feature_extractor.freeze_stats = True
        for _ in range(2):
            model.train()
            model.flat_parameters()[1].zero_()
            loss = model.review(inputs(), model(inputs()))['loss']
            loss.backward()
            losses.append(loss.item())
            assert all(torch.isfinite(p.grad).all() for p in model.parameters())
        assert losses[0] != losses[1]


def test_first_pass_under_capture_is_refused(monkeypatch):
    """The seed's copy from the host must not become a node of a graph."""
    from pb_sed_amd import engine, modules
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    rnn = modules.build_rnn(8, 64, 2, 4, 16, dropout=.5)
    with pytest.raises(RuntimeError, match='before a graph is captured'):
        engine.dropout_state(rnn, torch.device('cuda', 0))
    assert rnn.dropout_rng is None
