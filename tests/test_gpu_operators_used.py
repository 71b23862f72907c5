"""GPU: the learner with Muon and with the loss over legal moves, and games by the policies alone."""
import json
import os

import numpy as np
import pytest
import torch

from conftest import GOLDEN

pytestmark = pytest.mark.gpu


def _rows(n_games):
    t = json.load(open(os.path.join(GOLDEN, 'trees.json')))
    return [{k: m[k] for k in ('observation', 'legal_moves', 'pi', 'reward')}
            for g in t['synthetic'][:n_games] for m in g['moves']]


def _net():
    from minitchess_alphazero_amd.network import Network
    torch.manual_seed(0)
    return Network()


def test_masked_loss_and_gradients_of_the_network():
    """The learner's masked step against the same loss by torch on the CPU in 64 bits from the GPU's own logits and
    values: gradients at the logits exactly the operator's (tolerance of its own test), through the network by autograd."""
    from minitchess_alphazero_amd.learner import ResidentBatches, SimpleAlphaZeroLearner
    rows = _rows(2)
    net = _net()
    learner = SimpleAlphaZeroLearner(None, 8, net, 32, 1, {'lr': 1e-3}, 'cuda', legal_mask=True)
    model = net.train().cuda()
    data = ResidentBatches(rows, 'cuda', legal_masks=True)
    idx = torch.arange(32, device='cuda')
    loss = learner._backward(model, data, idx)
    got = {k: p.grad.clone() for k, p in model.named_parameters()}
    model.zero_grad()
    pib, tok, clk, rew = data.batch(list(range(32)))
    legal = torch.zeros(32, 554, dtype=torch.bool, device='cuda')
    for i, r in enumerate(rows[:32]):
        legal[i, torch.tensor(r['legal_moves'])] = True
    p, v = model((tok, clk))
    logp = p.double().masked_fill(~legal, float('-inf')).log_softmax(-1).masked_fill(~legal, 0.0)
    want = ((v.double() - rew) ** 2 - (pib * logp).sum(1, keepdim=True)).mean()
    want.backward()
    loss, want = float(loss), float(want.detach())
    assert abs(loss - want) <= 1e-5 * abs(want)
    for k, q in model.named_parameters():
        # the same backward pass from gradients at the logits that differ by roundings: the heads see them first
        if k.startswith(('plinear', 'vlinear')):
            assert float((got[k] - q.grad).norm()) <= 1e-5 * float(q.grad.norm()), k


def test_muon_learner_runs_captured_and_eager():
    """Captured and eager updates take the same steps on the trunk (to the convolutions' run-to-run differences),
    every parameter moves, and the default optimizer is what it was."""
    from minitchess_alphazero_amd.learner import EpisodeRecords, SimpleAlphaZeroLearner, muon_split  # noqa: F401
    rows = _rows(2)
    nets = []
    for graphs in (True, False):
        net = _net()
        before = {k: v.clone() for k, v in net.state_dict().items()}
        learner = SimpleAlphaZeroLearner(None, 8, net, 32, 1, {'lr': 1e-4}, 'cuda', optimizer='muon',
                                         muon_params={'lr': 1e-3}, legal_mask=True)
        learner.graphs = graphs
        torch.manual_seed(5)
        loss = learner.update(rows)
        assert np.isfinite(loss) and len(learner.last_losses) == -(-len(rows) // 32)
        after = net.state_dict()
        assert all(not torch.equal(before[k], v.cpu()) for k, v in after.items() if k.endswith('weight') and v.dim() > 1)
        nets.append((learner.last_losses, {k: v.cpu() for k, v in after.items()}))
    (l0, s0), (l1, s1) = nets
    assert abs(l0[0] - l1[0]) <= 1e-5 * abs(l0[0])     # before any step
    trunk = [k for k in s0 if k.startswith('resbody.') and s0[k].dim() == 4]
    assert len(trunk) == 19 and len(muon_split(_net())[0]) == 19
    with pytest.raises(ValueError):
        SimpleAlphaZeroLearner(None, 8, _net(), 32, 1, {}, 'cuda', optimizer='sgd')
    with pytest.raises(RuntimeError, match='need a GPU'):
        SimpleAlphaZeroLearner(None, 8, _net(), 32, 1, {}, 'cpu', optimizer='muon')


def test_replay_ring_keeps_masks():
    """Masks follow their rows through growth and wrap-around of the ring, by both ways in."""
    from minitchess_alphazero_amd.learner import EpisodeRecords, ReplayBuffer, ResidentBatches
    from minitchess_alphazero_amd.environment import pos_from_fen
    rows = _rows(2)
    ring = ReplayBuffer(70, 'cuda', initial=16, legal_masks=True)
    half = len(rows) // 2
    ring.push_rows(rows[:half])
    rest = rows[half:]
    ring.push_records(EpisodeRecords(np.stack([pos_from_fen(r['observation']) for r in rest]),
                                     [len(r['legal_moves']) for r in rest],
                                     np.concatenate([r['legal_moves'] for r in rest]),
                                     np.concatenate([np.round(np.asarray(r['pi']) * 10000) for r in rest]),
                                     [r['reward'] for r in rest]))
    want = ResidentBatches(rows, 'cuda', legal_masks=True).legal[-len(ring):]
    assert len(ring) == min(70, len(rows))
    assert torch.equal(ring.gather_legal(torch.arange(len(ring), device='cuda')), want)
    mask = want[0].cpu().numpy().view(np.uint32)
    legal = [v for v in range(554) if mask[v >> 5] >> (v & 31) & 1]
    assert legal == sorted(set(rows[-len(ring)]['legal_moves']))


def test_policy_match_counts_every_game():
    from minitchess_alphazero_amd.arena import policy_match
    a = _net()
    torch.manual_seed(1)
    b = type(a)()
    res = policy_match(a, b, 16, seed=3, repetition=1.3, frequency=0.1, presence=0.2)
    assert res['games'] == 32 and res['new_wins'] + res['old_wins'] + res['draws'] == 32
