"""GPU: orthogonalisation and the Muon step in the forms that large matrices take, against the definition in 64 bits.

Tolerances as in test_gpu_muon.py: TIGHT where all singular values lie within a factor of a few, LOOSE in general, plus half
a step of a 16-bit result.  Two steps joined form the second S as M S M, off by at most 12 (the square of 3.4445) times the
rounding 2^-22 of S in its small eigenvalues; 4.775 times that in M is 1.4e-5 relative in those directions a joined pair,
within LOOSE."""
import math

import pytest
import torch

from minitchess_alphazero_amd import optim
from test_gpu_muon import HALF, LOOSE, TIGHT, off, randn

pytestmark = pytest.mark.gpu


def reference(g, steps=5, eps=1e-7):
    """The definition in 64 bits, on the GPU, matrix by matrix."""
    if g.dim() == 3:
        return torch.stack([reference(m, steps, eps) for m in g])
    x = g.double()
    x = x / (x.square().sum().sqrt() + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    a, b, c = optim.COEFFICIENTS
    for _ in range(steps):
        s = x @ x.t().contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return (x.t() if tall else x).cpu()


def muon_reference(w, g, m, lr, momentum, nesterov, weight_decay):
    w, g, m = (t.double().flatten(1) for t in (w, g, m))
    m = momentum * m + (1 - momentum) * g
    u = (1 - momentum) * g + momentum * m if nesterov else m
    step = lr * math.sqrt(max(1.0, w.shape[0] / w.shape[1])) * reference(u)
    return (1 - lr * weight_decay) * w.cpu() - step, m.cpu(), step


# one matrix of 64-tiles, four of the trunk's of 128-tiles, tall, nearly square and ragged ones, tall of 128-tiles
@pytest.mark.parametrize('dtype', list(HALF), ids=str)
@pytest.mark.parametrize('nesterov', [True, False])
@pytest.mark.parametrize('n,shape', [(1, (256, 2304)), (4, (256, 256, 3, 3)), (1, (1000, 130)), (2, (300, 301)), (4, (1101, 500)),
                                     (2, (129, 3001)), (1, (800, 1300))], ids=str)
def test_muon_step(n, shape, nesterov, dtype):
    ws = [randn(*shape, seed=20 + i, dtype=dtype) for i in range(n)]
    gs = [randn(*shape, seed=30 + i, dtype=dtype) * 1e-2 for i in range(n)]
    ms = [randn(*shape, seed=40 + i) * 1e-2 for i in range(n)]
    args = dict(lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.05)
    want = [muon_reference(w, g, m, **args) for w, g, m in zip(ws, gs, ms)]
    optim.muon_step(ws, gs, ms, **args)
    for w, m, (w64, m64, step) in zip(ws, ms, want):
        assert off(m.view(m64.shape), m64) <= 8 * 2.0 ** -24
        bound = LOOSE * float(step.norm()) + (HALF[dtype] + 3 * 2.0 ** -24) * float(w64.norm())
        assert float((w.double().cpu().view(w64.shape) - w64).norm()) <= bound


@pytest.mark.parametrize('dtype', list(HALF), ids=str)
@pytest.mark.parametrize('shape,tight', [((3, 1021, 509), False), ((10, 896, 1000), False), ((1, 800, 1300), False),
                                         ((1, 1000, 1536), False), ((4, 1000, 1536), False), ((1, 256, 300), False), ((4, 1101, 500), False),
                                         ((2, 768, 3100), True), ((1, 5000, 1100), True)], ids=str)
def test_forms_of_the_products(shape, tight, dtype):
    g = randn(*shape, seed=sum(shape), dtype=dtype)
    assert off(optim.orthogonalize(g), reference(g)) <= (TIGHT if tight else LOOSE) + HALF[dtype]


@pytest.mark.parametrize('dtype', list(HALF), ids=str)
@pytest.mark.parametrize('shape', [(64, 3000), (150, 1100), (800, 1300), (1300, 800), (509, 1021), (1800, 2800)], ids=str)
@pytest.mark.parametrize('kind', ['low rank', 'falling'])
def test_small_singular_values(kind, shape, dtype):
    """A few strong directions and weak noise, or singular values falling over four decades: what two steps joined make of
    the small eigenvalues of S."""
    rank = 5 if kind == 'low rank' else min(shape)
    left = randn(shape[0], rank, seed=1) * torch.logspace(0, -4 if rank > 5 else 0, rank, device='cuda')
    g = left @ randn(rank, shape[1], seed=2)
    g = (g + 1e-2 * randn(*shape, seed=4) if rank == 5 else g).to(dtype)
    assert off(optim.orthogonalize(g), reference(g)) <= LOOSE + HALF[dtype]


@pytest.mark.parametrize('momentum', [0.9, 0.95, 0.999, 0.9999])
@pytest.mark.parametrize('shape', [(20, 60), (256, 2304)], ids=str)
def test_share_of_the_gradient_is_rounded_once(shape, momentum):
    """1 - momentum is taken in 64 bits: a momentum that starts at 0 is that share of the gradient, the share rounded to
    float and the product once more."""
    for nesterov in (True, False):
        w, g, m = randn(*shape, seed=1), randn(*shape, seed=2), torch.zeros(*shape, device='cuda')
        optim.muon_step([w], [g], [m], lr=0.1, momentum=momentum, nesterov=nesterov)
        want = (1 - momentum) * g.double()
        assert bool(((m.double() - want).abs() <= 2.0 * 2.0 ** -24 * want.abs() * (1 + 2.0 ** -20)).all())
