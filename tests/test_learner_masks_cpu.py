"""CPU: the learner's legal masks are the rows' own legal lists."""
import numpy as np
import torch

from minitchess_alphazero_amd import _lib
from minitchess_alphazero_amd.environment import pos_from_fen, pos_legal
from minitchess_alphazero_amd.learner import EpisodeRecords, ResidentBatches

START = '2nbk/2ppp/5/5/PPP2/KBN2 w 0 1'


def unpack(masks):
    words = masks.numpy().view(np.uint32)
    return [[v for v in range(554) if m[v >> 5] >> (v & 31) & 1] for m in words]


def test_masks_follow_the_rules_of_the_rows():
    """Games with double pawn steps: a mask by the default rules would cut those moves, and their targets, off."""
    legal = [int(c) for c in pos_legal(pos_from_fen(START), _lib.RF_DEFAULT | _lib.RF_DOUBLE_STEP)]
    assert set(legal) > set(int(c) for c in pos_legal(pos_from_fen(START)))
    rows = [{'observation': START, 'legal_moves': moves, 'pi': [1 / len(moves)] * len(moves), 'reward': 1.0}
            for moves in (legal, legal[:1], [3, 3, 0, 553, 31, 32], legal)]
    want = [sorted(set(r['legal_moves'])) for r in rows]
    data = ResidentBatches(rows, 'cpu', legal_masks=True)
    assert unpack(data.legal) == want
    assert unpack(data.gather_legal(torch.tensor([2, 0]))) == [want[2], want[0]]
    records = EpisodeRecords(np.stack([pos_from_fen(START)] * 4), [len(r['legal_moves']) for r in rows],
                             np.concatenate([r['legal_moves'] for r in rows]), np.ones(sum(len(r['legal_moves']) for r in rows)),
                             np.ones(4))
    assert unpack(ResidentBatches(records, 'cpu', legal_masks=True).legal) == want
    assert ResidentBatches([rows[0]], 'cpu').legal is None


def test_many_rows():
    from minitchess_alphazero_amd.learner import _masks_of
    g = np.random.default_rng(0)
    k = torch.from_numpy(g.integers(0, 4, 70000))
    codes = torch.from_numpy(g.integers(0, 554, int(k.sum())).astype(np.int16))
    masks = _masks_of(k, codes).numpy().view(np.uint32)
    e = np.concatenate([[0], np.cumsum(k.numpy())])
    for i in (0, 1, 32766, 32767, 32768, 32769, 65536, 69999):
        assert unpack(torch.from_numpy(masks[i:i + 1].view(np.int32)))[0] == sorted(set(codes[e[i]:e[i + 1]].tolist()))
