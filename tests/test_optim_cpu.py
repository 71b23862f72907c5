"""CPU: what Muon and the learner's options refuse or compute on the host."""
import pytest
import torch

from minitchess_alphazero_amd import optim


def test_first_step_is_not_captured(monkeypatch):
    """A captured first step would set its momenta to 0 in every replay."""
    p = torch.nn.Parameter(torch.randn(4, 8))
    opt = optim.Muon([p])
    p.grad = torch.randn(4, 8)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    with pytest.raises(RuntimeError, match='before the capture'):
        opt.step()
    assert not opt.state[p]
    opt.state[p]['momentum_buffer'] = torch.zeros(4, 8)
    with pytest.raises(ValueError, match='GPU'):        # a later step goes on to the kernels
        opt.step()
