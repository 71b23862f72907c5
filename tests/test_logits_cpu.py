"""CPU: what the logits operators make of their arguments before they call a kernel."""
import ctypes

import pytest
import torch

from minitchess_alphazero_amd import _lib
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


BUF = ctypes.create_string_buffer(8192)
P = (ctypes.addressof(BUF) + 255) // 256 * 256
PEN = (ctypes.c_double * 3)(1.2, 0.1, 0.1)


def refused(rc, why):
    assert rc == _lib.E_FAIL
    assert why in _lib.lib().mtaz_last_error().decode()


# [2][40] float32 at P: 320 bytes
@pytest.mark.parametrize('legal,bias,bias_stride,actions,lengths,per_row', [
    (P + 316, None, 0, None, None, None),                       # its first word is the output's last element
    (P + 1024, P, 0, None, None, None),                         # one bias for both rows, where the first row is written
    (P + 1024, P, 41, None, None, None),
    (P + 1024, P + 4, 40, None, None, None),
    (None, None, 0, P + 304, None, None), (None, None, 0, P - 16, None, None), (None, None, 0, P + 1024, P + 160, None),
    (None, None, 0, P + 1024, None, P + 300)])
def test_output_over_what_other_rows_read_is_refused(legal, bias, bias_stride, actions, lengths, per_row):
    L = _lib.lib()
    refused(L.mtaz_adjust_logits(0, 2, 40, 0, P + 2048, 40, P, 40, legal, 2, bias, bias_stride, actions, 4, 4 if actions else 0,
                                 lengths, PEN, per_row, None), 'overlaps the mask, the bias or the actions')
    if bias is None:
        for grads in ((P, 40, None, 0), (None, 0, P, 40), (None, 0, P, 0)):
            hit = grads[3] != 0 or grads[0] is not None or (P <= (actions or 0) < P + 160)
            if hit:
                refused(L.mtaz_adjust_logits_grad(0, 2, 40, 0, P + 2048, 40, P + 3072, 40, *grads, legal, 2, actions, 4,
                                                  4 if actions else 0, lengths, PEN, per_row, P + 4096, 1024, None),
                        'overlaps the mask or the actions')
    if legal is not None and bias is None:
        refused(L.mtaz_policy_loss(0, 2, 40, 0, 0, P + 2048, 40, P + 3072, 40, legal, 2, None, None, P + 4096, P + 4352, P, 40,
                                   None, 1.0, P + 4608, 256, None), 'overlaps the mask')


def test_workspaces_off_their_boundary_are_refused():
    L = _lib.lib()
    for off in (4, 16, 128):
        refused(L.mtaz_policy_loss(0, 2, 40, 0, 0, P, 40, P + 1024, 40, None, 0, None, None, P + 2048, P + 2304, None, 0, None, 1.0,
                                   P + 4096 + off, 1024, None), 'aligned')
        refused(L.mtaz_adjust_logits_grad(0, 2, 40, 0, P, 40, None, 0, P + 1024, 40, P + 2048, 0, None, 0, None, 0, 0, None, None,
                                          None, P + 4096 + off, 1024, None), 'aligned')


def test_rows_that_a_launch_does_not_hold_are_refused():
    """2^26 - 4 waves of 64 threads, four a workgroup, are the most below 2^32 threads."""
    L, most = _lib.lib(), (1 << 26) - 4
    assert L.mtaz_policy_loss_workspace(most, 40) == 256
    for rows in (most + 1, most + 3, most + 4):
        refused(L.mtaz_policy_loss_workspace(rows, 40), 'too many rows')
    assert L.mtaz_adjust_logits_grad_workspace(most, 40) > 0
    for rows, history in ((most // 2 + 1, 65), (most // 4 + 1, 256)):
        refused(L.mtaz_adjust_logits_grad(0, rows, 1, 0, P, 1, P + 1024, 1, P + 2048, 1, None, 0, None, 0, P + 4096, 0, history, None,
                                          PEN, None, None, 0, None), 'too many rows')


def test_histories_past_an_int_are_refused():
    """2^32 + 5 entries a row (one entry, expanded) would be 5 where they are counted in 32 bits."""
    x = torch.zeros(2, 40)
    for entries in (1 << 32) + 5, (1 << 31) + 1, (1 << 30) + 1:
        with pytest.raises(ValueError, match='at most 2'):
            ops._Taken(x, torch.zeros(1, 1, dtype=torch.int32).expand(2, entries), None, 1.2, 0.0, 0.0)
    refused(_lib.lib().mtaz_adjust_logits(0, 2, 40, 0, P, 40, P + 1024, 40, None, 0, None, 0, P + 2048, 0, (1 << 30) + 1, None, PEN,
                                          None, None), 'history')
