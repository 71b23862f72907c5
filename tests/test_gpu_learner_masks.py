"""GPU: the replay ring's legal masks are the rows' own legal lists, by every way in."""
import numpy as np
import pytest
import torch

from minitchess_alphazero_amd import _lib
from minitchess_alphazero_amd.environment import pos_from_fen, pos_legal
from test_learner_masks_cpu import START, unpack

pytestmark = pytest.mark.gpu


def test_ring_follows_the_rules_of_the_rows():
    from minitchess_alphazero_amd.learner import EpisodeRecords, ReplayBuffer, ResidentBatches
    legal = [int(c) for c in pos_legal(pos_from_fen(START), _lib.RF_DEFAULT | _lib.RF_DOUBLE_STEP)]
    rows = [{'observation': START, 'legal_moves': legal[i % 3:], 'pi': [1 / len(legal[i % 3:])] * len(legal[i % 3:]), 'reward': 0.0}
            for i in range(11)]
    want = [sorted(set(r['legal_moves'])) for r in rows]
    records = EpisodeRecords(np.stack([pos_from_fen(START)] * 11), [len(r['legal_moves']) for r in rows],
                             np.concatenate([r['legal_moves'] for r in rows]), np.ones(sum(len(r['legal_moves']) for r in rows)),
                             np.zeros(11))
    assert unpack(ResidentBatches(rows, 'cuda', legal_masks=True).legal.cpu()) == want
    for size in (30, 7):                    # more rows than the ring holds: the newest stay
        for first, second in ((rows, records), (records, rows)):
            ring = ReplayBuffer(size, 'cuda', initial=4, legal_masks=True)
            for part in (first, second):
                (ring.push_rows if part is rows else ring.push_records)(part)
            got = unpack(ring.gather_legal(torch.arange(len(ring), device='cuda')).cpu())
            assert got == (want + want)[-size:]


@pytest.mark.parametrize('options', [{}, {'optimizer': 'muon', 'muon_params': {'lr': 1e-3}, 'legal_mask': True}], ids=['adamw', 'muon'])
def test_captured_gradients_stay_alive_past_a_partial_batch(options):
    """A partial batch runs between replays of the captured step, which writes to the gradients that it was captured
    with: they must be the parameters' own to the end."""
    from minitchess_alphazero_amd.learner import SimpleAlphaZeroLearner
    from test_gpu_operators_used import _net, _rows
    rows = _rows(1)
    rows = rows[:len(rows) // 8 * 8 + 3]
    assert len(rows) % 8 == 3
    held = {}

    class Learner(SimpleAlphaZeroLearner):
        def _graph_step(self, model, optimizer, data):
            step = super()._graph_step(model, optimizer, data)
            held.update({n: p.grad for n, p in model.named_parameters()})
            return step
    net = _net()
    learner = Learner(None, 8, net, 8, 2, {'lr': 1e-4}, 'cuda', **options)
    learner.update(rows)
    assert len(held) == len(list(net.parameters())) and len(learner.last_losses) == 2 * -(-len(rows) // 8)
    assert all(p.grad is held[n] or p.grad.data_ptr() == held[n].data_ptr() for n, p in net.named_parameters())
    assert np.isfinite(learner.last_losses).all()
