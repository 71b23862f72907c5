"""CPU: what Muon and the learner's options refuse or compute on the host."""
import pytest
import torch

from minitchess_alphazero_amd import _lib, optim


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


def test_a_refused_step_has_changed_nothing(monkeypatch):
    """All shapes are looked at before the first group's kernels are called."""
    called = []

    class Library:
        def __getattr__(self, name):
            return (lambda *args: called.append(name) or 0) if name == 'mtaz_muon_step' else getattr(real, name)
    real = _lib.lib()
    monkeypatch.setattr(_lib, 'lib', lambda: Library())
    monkeypatch.setattr(optim, '_stream', lambda device: 0)
    monkeypatch.setattr(optim, '_check_type', lambda t, what: None)

    def tensors(*shapes):
        return [torch.zeros(s) for s in shapes]
    ok, bad = (8, 16), (70000, 2)
    with pytest.raises(_lib.MtazError, match='rows and cols'):
        optim.muon_step(tensors(ok, bad), tensors(ok, bad), tensors(ok, bad), lr=0.1)
    assert not called
    optim.muon_step(tensors(ok, ok[::-1]), tensors(ok, ok[::-1]), tensors(ok, ok[::-1]), lr=0.1)
    assert called == ['mtaz_muon_step'] * 2
