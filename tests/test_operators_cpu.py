"""CPU: refusals of the learner operators' C entries (their checks come before any device call) and of the Python
layer for tensors that are not on a GPU."""
import ctypes

import pytest
import torch

from minitchess_alphazero_amd import _lib, logits, optim

BUF = ctypes.create_string_buffer(4096)
P = (ctypes.addressof(BUF) + 255) // 256 * 256
CO = (ctypes.c_double * 3)(*optim.COEFFICIENTS)
ONE = (ctypes.c_void_p * 1)(P)
PEN = (ctypes.c_double * 3)(1.2, 0.1, 0.1)


def refused(rc, why):
    assert rc == _lib.E_FAIL
    assert why in _lib.lib().mtaz_last_error().decode()


def ortho(n=1, rows=4, cols=8, dtype=0, grad=ONE, out=ONE, steps=5, co=CO, eps=1e-7, work=P, size=1 << 40):
    return _lib.lib().mtaz_orthogonalize(0, n, rows, cols, dtype, grad, out, steps, co, eps, work, size, None)


@pytest.mark.parametrize('args,why', [
    (dict(n=-1), 'n must not'), (dict(rows=0), 'rows and cols'), (dict(cols=65537), 'rows and cols'),
    (dict(rows=40000, cols=40000), 'rows and cols'), (dict(dtype=3), 'element type'), (dict(steps=0), 'steps'),
    (dict(steps=33), 'steps'), (dict(eps=-1.0), 'eps'), (dict(eps=float('nan')), 'eps'),
    (dict(co=(ctypes.c_double * 3)(float('inf'), 0, 0)), 'finite'), (dict(co=(ctypes.c_double * 3)(30, 0, 0)), 'singular values'),
    (dict(grad=(ctypes.c_void_p * 1)(None)), 'null matrix'), (dict(grad=None), 'no matrices'), (dict(size=100), 'workspace'),
    (dict(work=P + 16), 'workspace'), (dict(work=None), 'workspace')])
def test_orthogonalize_refuses(args, why):
    refused(ortho(**args), why)


def test_orthogonalize_sizes():
    L = _lib.lib()
    assert ortho(n=0) == 0
    one, two = (L.mtaz_orthogonalize_workspace(n, 100, 300, 0) for n in (1, 2))
    assert 0 < one < two <= 2 * one
    assert L.mtaz_orthogonalize_workspace(64, 100, 300, 0) == L.mtaz_orthogonalize_workspace(1000, 100, 300, 0)
    assert L.mtaz_orthogonalize_workspace(1, 0, 300, 0) == _lib.E_FAIL


@pytest.mark.parametrize('momentum,lr,why', [(1.0, 0.1, 'momentum'), (-0.1, 0.1, 'momentum'), (float('nan'), 0.1, 'momentum'),
                                             (0.9, float('inf'), 'finite')])
def test_muon_refuses(momentum, lr, why):
    refused(_lib.lib().mtaz_muon_step(0, 1, 4, 8, 0, ONE, ONE, ONE, lr, momentum, 1, 0.0, 1.0, 5, CO, 1e-7, P, 1 << 40,
                                      None), why)


def adjust(rows=2, cols=40, dtype=0, x=P, xs=40, out=P, os=40, actions=P, stride=4, history=4, pen=PEN, per_row=None):
    return _lib.lib().mtaz_adjust_logits(0, rows, cols, dtype, x, xs, out, os, None, 0, None, 0, actions, stride, history,
                                         None, pen, per_row, None)


@pytest.mark.parametrize('args,why', [
    (dict(rows=-1), 'rows'), (dict(cols=0), 'cols'), (dict(cols=(1 << 24) + 1), 'cols'), (dict(rows=1 << 31), 'too many rows'),
    (dict(dtype=-1), 'element type'), (dict(x=None), 'no logits'), (dict(os=39), 'overlap'), (dict(xs=41), 'in place'),
    (dict(history=-1), 'history'), (dict(pen=None), 'without penalties'), (dict(stride=-1), 'stride'),
    (dict(pen=(ctypes.c_double * 3)(0, 0, 0)), 'positive')])
def test_adjust_refuses(args, why):
    refused(adjust(**args), why)


def test_adjust_nothing():
    assert adjust(rows=0) == 0


@pytest.mark.parametrize('args,why', [
    (dict(gy=None), 'incoming'), (dict(x=None), 'needs the logits'), (dict(gs=39), 'overlap'), (dict(bs=39), 'overlap'),
    (dict(bs=0, size=100), 'workspace'), (dict(bs=0, work=None), 'workspace'), (dict(), 'in place')])
def test_adjust_grad_refuses(args, why):
    a = dict(gy=P, x=P, gs=40, bs=40, work=P, size=1 << 20)
    a.update(args)
    refused(_lib.lib().mtaz_adjust_logits_grad(0, 2, 40, 0, a['gy'], 40, a['x'], 40, P, a['gs'], P, a['bs'], None, 0, P, 4, 4,
                                               None, PEN, None, a['work'], a['size'], None), why)


@pytest.mark.parametrize('args,why', [
    (dict(rows=0), 'no rows'), (dict(target=2), 'targets are'), (dict(z=None), 'no logits'), (dict(stats=None), 'statistics'),
    (dict(value=None), 'without'), (dict(reward=None), 'without'), (dict(value=None, reward=None), 'not there'),
    (dict(gs=39), 'overlap'), (dict(loss=None), 'place for'), (dict(size=8), 'workspace')])
def test_loss_refuses(args, why):
    a = dict(rows=2, target=0, z=P, stats=P, value=P, reward=P, gs=40, loss=P, size=1 << 20)
    a.update(args)
    refused(_lib.lib().mtaz_policy_loss(0, a['rows'], 40, 1, a['target'], a['z'], 40, P, 40, None, 0, a['value'], a['reward'],
                                        a['loss'], a['stats'], P, a['gs'], P, 1.0, P, a['size'], None), why)


def test_loss_grad_refuses():
    f = _lib.lib().mtaz_policy_loss_grad
    refused(f(0, 2, 40, 0, 0, P, 40, P, 40, None, 0, None, None, P, None, P, 40, None, None), 'incoming')
    assert f(0, 2, 40, 0, 0, P, 40, P, 40, None, 0, None, None, P, P, None, 40, None, None) == 0


@pytest.mark.parametrize('x,xs,out,os,rows,why', [
    (P + 4, 40, P, 40, 2, 'overlaps'), (P, 40, P + 4 * 79, 40, 2, 'overlaps'), (P, 80, P + 4 * 39, 80, 2, 'overlaps'),
    (P, 80, P + 4 * 41, 80, 2, 'overlaps'), (P, 0, P, 40, 2, 'in place'), (P, 40, P, 41, 2, 'in place'),
    (P, 41, P, 40, 1 << 25, 'too many rows')])
def test_overlaps_and_sizes_refused(x, xs, out, os, rows, why):
    cols = 40 if rows < 1 << 25 else 2049
    refused(adjust(x=x, xs=xs, out=out, os=max(os, cols), cols=cols, rows=rows, actions=None), why)


def test_loss_gradient_over_the_logits_refused():
    L = _lib.lib()

    def loss(z, zs, grad, gs, dtype=1, target=P + 1600, ttype=1):
        return L.mtaz_policy_loss(0, 2, 40, dtype, ttype, z, zs, target, 40, None, 0, None, None, P, P + 1024, grad, gs, None, 1.0,
                                  P, 0, None)
    refused(loss(P, 40, P + 2, 40), 'workspace')          # the other checks come first
    for z, zs, grad, gs, ttype in ((P, 40, P + 2, 40, 1), (P, 41, P, 40, 1), (P, 40, P + 1600, 40, 0), (P, 40, P + 1598, 40, 1)):
        refused(L.mtaz_policy_loss(0, 2, 40, 1, ttype, z, zs, P + 1600, 40, None, 0, None, None, P, P + 1024, grad, gs, None, 1.0,
                                   P, 256, None), 'not in place')


def test_workspace_of_large_matrices_does_not_grow():
    """Matrices that fill the chip one by one go through the kernels one after the other."""
    one, many = (_lib.lib().mtaz_orthogonalize_workspace(n, 16384, 16384, 2) for n in (1, 50))
    assert one == many
    assert _lib.lib().mtaz_orthogonalize_workspace(64, 4096, 4096, 0) < 3 << 30


def test_python_refuses_cpu_tensors():
    g = torch.randn(4, 8)
    for call in (lambda: optim.orthogonalize(g), lambda: optim.muon_step([g], [g], [g.clone()], lr=0.1),
                 lambda: logits.adjust_logits(g), lambda: logits.policy_value_loss(g, g),
                 lambda: logits.policy_value_loss_grad(g, g)):
        with pytest.raises(ValueError, match='GPU'):
            call()
    with pytest.raises(ValueError, match='two dimensions'):
        optim.Muon([torch.nn.Parameter(torch.zeros(5))])
    with pytest.raises(ValueError, match='momentum'):
        optim.Muon([torch.nn.Parameter(torch.zeros(5, 5))], momentum=1.5)
    with pytest.raises(ValueError, match='1 parameters, 0 gradients'):
        optim.muon_step([g], [], [], lr=0.1)
