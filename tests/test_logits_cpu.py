"""CPU: what the logits operators make of their arguments before they call a kernel."""
import pytest
import torch

from minitchess_alphazero_amd import logits as ops


def test_penalties_are_float32_under_another_default_type():
    x, actions = torch.zeros(2, 5), torch.zeros(2, 3, dtype=torch.int32)
    rep = torch.full((2,), 1.5)
    before = torch.get_default_dtype()
    for default in (torch.float64, torch.bfloat16, torch.float32):
        torch.set_default_dtype(default)
        try:
            taken = ops._Taken(x, actions, None, rep, 0.25, 0.5)
        finally:
            torch.set_default_dtype(before)
        assert taken.tensors[2].dtype == torch.float32
        assert torch.equal(taken.tensors[2], torch.tensor([[1.5, 0.25, 0.5]] * 2))
