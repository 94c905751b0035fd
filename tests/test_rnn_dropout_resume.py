"""The masks between GRU layers go on from a trainer checkpoint (pb_sed_amd.engine.dropout_state, trainer.Trainer)."""
import os
import socket
import sys

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CPU = torch.device('cpu')


def build(dropout=.2):
    from pb_sed_amd.models import weak_label
    from pb_sed_amd.trainer import Trainer
    net = dict(out_channels_2d=[16, 16, 32], pool_sizes_2d=[1, (2, 1), (2, 1)], kernel_size_2d=3, out_channels_1d=[64, 64], kernel_size_1d=[1, 3])
    model = weak_label.CRNN.build(num_events=10, hidden_size=64, num_layers=2, net=net, rnn_dropout=dropout)
    return model, Trainer(model)


def passes(model, n):
    """The (seed, step) of n training passes of both networks."""
    from pb_sed_amd import engine, ops
    import numpy as np
    keep = ops.host_to_device
    ops.host_to_device = lambda a, device, dtype=None: torch.from_numpy(np.array(a)).to(dtype)
    try:
        return [engine.dropout_state(w, CPU).tolist() for _ in range(n) for w in (model.rnn_fwd, model.rnn_bwd)]
    finally:
        ops.host_to_device = keep


def test_a_resumed_run_draws_the_masks_of_the_run_that_went_on(tmp_path):
    torch.manual_seed(5)
    model, tr = build()
    first = passes(model, 3)
    path = tr.save_checkpoint(str(tmp_path))
    on = passes(model, 2)
    torch.manual_seed(6)
    model2, tr2 = build()
    tr2.load_checkpoint(path)
    assert passes(model2, 2) == on and on[0][0] == first[0][0] and on[0][1] == 3
    # a file from before a first pass, or without the entry: the seed is drawn
    model3, tr3 = build()
    path = tr3.save_checkpoint(str(tmp_path), 'new.pth')
    model4, tr4 = build()
    tr4.load_checkpoint(path)
    assert model4.rnn_fwd.dropout_rng is None
    ckpt = tr.state_dict()
    del ckpt['rnn_dropout']
    tr4.load_state_dict(ckpt)
    assert model4.rnn_fwd.dropout_rng is None and len(passes(model4, 1)) == 2
    # without dropout there is nothing to carry
    assert build(0.)[1].state_dict()['rnn_dropout'] == {}


def _worker(rank, world, port, out):
    sys.path.insert(0, ROOT)
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port))
    dist.init_process_group('gloo', rank=rank, world_size=world)
    torch.manual_seed(0)
    model, tr = build()
    torch.manual_seed(10 + rank)
    passes(model, 2)
    path = tr.save_checkpoint(out)
    dist.barrier()
    on = passes(model, 1)
    model2, tr2 = build()
    tr2.load_checkpoint(path)
    ok = passes(model2, 1) == on
    with open(os.path.join(out, f'ok{rank}'), 'w') as f:
        f.write(f'{ok} {on[0][0]}')
    dist.destroy_process_group()


def test_every_rank_goes_on_with_its_own_masks(tmp_path):
    with socket.socket() as s:
        s.bind(('127.0.0.1', 0))
        port = s.getsockname()[1]
    mp.spawn(_worker, args=(2, port, str(tmp_path)), nprocs=2, join=True)
    got = [open(tmp_path / f'ok{r}').read().split() for r in range(2)]
    assert [g[0] for g in got] == ['True', 'True'] and got[0][1] != got[1][1]
