"""GPU: orthogonalize, muon_step and Muon against the definition in 64 bits.

Tolerances (relative 2-norm).  A plane pair (hi, lo) holds 22 bits: a value is off by at most 2^-23 of itself.  A
Newton-Schulz step rounds X, S and B (|b S + c S S| <= 2.9 while X' ~ 1), so it adds at most about
(1 + 2 * 2.9 + 1) 2^-23 < 2^-20.  Where all singular values lie within a factor of a few (a Gaussian matrix
with one side at least 4 times the other), error and result grow together and five steps stay below
10 * 2^-20 < 1e-5.  In general, error of the first steps in directions of tiny singular values grows by up to
3.4445 a step against a result that does not: (1 + 3.4 + 11.9 + 40.9 + 140.8) 2^-20 < 2e-4.  A 16-bit result
adds half a step of its type."""
import math

import pytest
import torch

from minitchess_alphazero_amd import _lib, optim

pytestmark = pytest.mark.gpu
TIGHT, LOOSE = 1e-5, 2e-4
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def reference(g, steps=5, co=optim.COEFFICIENTS, eps=1e-7):
    x = g.double().cpu()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(steps):
        s = x @ x.mT
        x = co[0] * x + (co[1] * s + co[2] * (s @ s)) @ x
    return x.mT if tall else x


def off(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize('dtype', list(HALF), ids=str)
@pytest.mark.parametrize('shape', [(1, 4, 16), (3, 61, 554), (2, 554, 61), (1, 64, 256), (2, 65, 257), (1, 256, 72),
                                   (5, 256, 2304), (1, 129, 1000), (2, 1000, 130)], ids=str)
def test_gaussian(shape, dtype):
    g = randn(*shape, seed=sum(shape), dtype=dtype)
    assert off(optim.orthogonalize(g), reference(g)) <= TIGHT + HALF[dtype]


@pytest.mark.parametrize('shape,dtype', [((8, 530, 1100), torch.float32), ((1, 1450, 2900), torch.bfloat16),
                                         ((67, 140, 300), torch.float32)], ids=str)
def test_other_tiles_and_groups(shape, dtype):
    g = randn(*shape, seed=sum(shape), dtype=dtype)
    assert off(optim.orthogonalize(g), reference(g)) <= TIGHT + HALF[dtype]


@pytest.mark.parametrize('shape', [(1, 1), (1, 7), (7, 1), (2, 2), (31, 33), (64, 64), (128, 128), (255, 255), (300, 301)],
                         ids=str)
def test_square_small_and_odd(shape):
    g = randn(*shape, seed=3)
    assert off(optim.orthogonalize(g), reference(g)) <= LOOSE


@pytest.mark.parametrize('shape', [(4133, 15), (5, 9000), (64, 3000), (150, 1100)], ids=str)
def test_long_sides_keep_32_bits(shape):
    """A few strong directions and noise: within twice of what the same steps in float give (sums of r and L terms,
    errors of both sides alike in kind)."""
    g = randn(*shape, seed=sum(shape)).cpu()
    u = randn(shape[0], 1, seed=1).cpu() @ randn(1, shape[1], seed=2).cpu()
    g = (u + 0.3 * g).cuda()
    want = reference(g)
    x = g.cpu() / g.cpu().norm()
    x = x.mT if shape[0] > shape[1] else x
    a, b, c = optim.COEFFICIENTS
    for _ in range(5):
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    plain = off(x.mT if shape[0] > shape[1] else x, want)
    assert off(optim.orthogonalize(g), want) <= 2 * plain


@pytest.mark.parametrize('shape', [(96, 400), (700, 90)], ids=str)
def test_low_rank(shape):
    g = randn(shape[0], 5, seed=1) @ randn(5, shape[1], seed=2) + 1e-2 * randn(*shape, seed=4)
    got, want = optim.orthogonalize(g), reference(g)
    assert off(got, want) <= LOOSE
    # the noise's singular values are some 2.3e-4 of the norm: five steps take them to 3.4445^5 = 485 times that, 0.11,
    # not to 1; they differ from the definition's by at most the difference's norm
    s, w = (torch.linalg.svdvals(t) for t in (got.double().cpu(), want))
    assert float(s.max()) < 1.3 and float((s - w).abs().max()) <= LOOSE * float(want.norm())


@pytest.mark.parametrize('steps,co', [(1, (2.0, -1.5, 0.5)), (3, (1.5, -0.5, 0.0)), (12, (15 / 8, -10 / 8, 3 / 8))])
def test_other_steps_and_coefficients(steps, co):
    g = randn(40, 200, seed=7)
    assert off(optim.orthogonalize(g, steps=steps, coefficients=co), reference(g, steps, co)) <= LOOSE


@pytest.mark.parametrize('factor', [1e30, 1e-18, 1e-30], ids=str)
def test_range_of_gradients(factor):
    """The norm is summed in 64 bits: squares of 1e30 and 1e-30 are in range; eps 0 divides by the norm alone."""
    g = randn(33, 150, seed=5) * factor
    assert off(optim.orthogonalize(g, eps=0.0), reference(g, eps=0.0)) <= TIGHT


def test_zeros_nan_and_neighbours():
    g = randn(4, 20, 90, seed=6)
    want = reference(g)
    g[1] = 0
    g[2, 3, 4] = math.nan
    got = optim.orthogonalize(g)
    assert not got[1].any() and got[2].isnan().any()
    for i in (0, 3):
        assert off(got[i], want[i]) <= TIGHT


@pytest.mark.parametrize('shape', [(5, 24), (17, 40), (61, 300), (100, 130), (3, 2000), (200, 300)], ids=str)
def test_nothing_is_left_from_another_matrix(shape):
    """Matrices of NaN on every CU before: what they leave in LDS must not get into padded rows and columns."""
    optim.orthogonalize(torch.full((1024, 96, 96), math.nan, device='cuda'))
    g = randn(2, *shape, seed=12)
    assert off(optim.orthogonalize(g), reference(g)) <= LOOSE


def test_many_matrices_in_groups():
    g = randn(131, 5, 24, seed=8)           # two launches of 64 and one of 3
    got = optim.orthogonalize(g)
    assert off(got, reference(g)) <= TIGHT
    assert torch.equal(optim.orthogonalize(g[70:71]), got[70:71])
    assert optim.orthogonalize(g[:0]).shape == (0, 5, 24)


def test_layouts_out_and_repeatability():
    base = randn(3, 80, 48, seed=9)
    g = base.mT                             # strides (., 1, 48)
    want = optim.orthogonalize(g.contiguous())
    assert torch.equal(optim.orthogonalize(g), want)
    work = g.contiguous()
    assert optim.orthogonalize(work, out=work) is work and torch.equal(work, want)
    odd = torch.empty(3 * 48 * 80 + 1, device='cuda')[1:].view(3, 48, 80)   # 4-byte aligned only
    odd.copy_(g)
    out = torch.empty(3 * 48 * 80 + 1, device='cuda')[1:].view(3, 48, 80)
    optim.orthogonalize(odd, out=out)
    assert torch.equal(out, want)


def test_two_streams_at_once():
    g = [randn(2, 100, 700, seed=s) for s in (10, 11)]
    want = [optim.orthogonalize(x) for x in g]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in g]
    got = [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(optim.orthogonalize(g[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(x, want[k]) for x in got[k])


def _muon_reference(ws, gs, ms, lr, momentum, nesterov, weight_decay, scale=None):
    out = []
    for w, g, m in zip(ws, gs, ms):
        rows = w.shape[0]
        w64, g64 = w.double().cpu().view(rows, -1), g.double().cpu().reshape(rows, -1)
        m64 = momentum * m.double().cpu().view(rows, -1) + (1 - momentum) * g64
        u = (1 - momentum) * g64 + momentum * m64 if nesterov else m64
        f = math.sqrt(max(1.0, rows / w64.shape[1])) if scale is None else scale
        step = lr * f * reference(u)
        out.append(((1 - lr * weight_decay) * w64 - step, m64, step))
    return out


@pytest.mark.parametrize('dtype', list(HALF), ids=str)
@pytest.mark.parametrize('nesterov', [True, False])
def test_muon_step(dtype, nesterov):
    """Shapes of one type go together, conv weights as [out, in * kh * kw]; the momentum is float32."""
    shapes = [(16, 8, 3, 3), (16, 8, 3, 3), (100, 20), (16, 8, 3, 3), (3, 200)]
    ws = [randn(*s, seed=20 + i, dtype=dtype) for i, s in enumerate(shapes)]
    gs = [randn(*s, seed=30 + i, dtype=dtype) * 1e-2 for i, s in enumerate(shapes)]
    ms = [randn(*s, seed=40 + i) * 1e-2 for i, s in enumerate(shapes)]
    args = dict(lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.05)
    want = _muon_reference(ws, gs, ms, **args)
    optim.muon_step(ws, gs, ms, **args)
    for w, m, (w64, m64, step) in zip(ws, ms, want):
        # the fused multiply-add of the momentum and its coefficients: four roundings of 2^-24, of sums at most
        # twice the result's size in norm; the weight: two roundings in float and one to its type
        assert off(m.view(m64.shape), m64) <= 8 * 2.0 ** -24
        bound = LOOSE * float(step.norm()) + (HALF[dtype] + 3 * 2.0 ** -24) * float(w64.norm())
        assert float((w.double().cpu().view(w64.shape) - w64).norm()) <= bound


def test_muon_optimizer_matches_steps_and_restores():
    torch.manual_seed(0)
    a = torch.nn.Parameter(randn(24, 90, seed=50, dtype=torch.bfloat16))
    b = torch.nn.Parameter(a.detach().clone())
    opt = optim.Muon([a], lr=0.05, weight_decay=0.01)
    m = torch.zeros(24, 90, device='cuda')
    for t in range(3):
        a.grad = randn(24, 90, seed=60 + t, dtype=torch.bfloat16)
        v = a._version
        opt.step()
        assert a._version > v
        optim.muon_step([b.data], [a.grad], [m], lr=0.05, weight_decay=0.01)
    assert torch.equal(a, b) and torch.equal(opt.state[a]['momentum_buffer'], m)
    other = optim.Muon([torch.nn.Parameter(b.detach().clone())], lr=1.0)
    other.load_state_dict(opt.state_dict())
    p = other.param_groups[0]['params'][0]
    assert other.state[p]['momentum_buffer'].dtype == torch.float32
    a.grad = randn(24, 90, seed=70, dtype=torch.bfloat16)
    p.grad = a.grad.clone()
    opt.step(), other.step()
    assert torch.equal(p, a)


def test_captured_steps_replay():
    """One step captured and replayed, with eager steps of other parameters between the replays."""
    w, g, m = randn(32, 144, seed=80), randn(32, 144, seed=81), torch.zeros(32, 144, device='cuda')
    ref = [t.clone() for t in (w, m)]
    other = [randn(32, 144, seed=82), randn(32, 144, seed=83), torch.zeros(32, 144, device='cuda')]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        optim.muon_step([other[0]], [other[1]], [other[2]], lr=0.1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optim.muon_step([w], [g], [m], lr=0.1)
    for t in range(4):
        g.copy_(randn(32, 144, seed=90 + t))
        graph.replay()
        optim.muon_step([other[0]], [other[1]], [other[2]], lr=0.1)
        optim.muon_step([ref[0]], [g], [ref[1]], lr=0.1)
        torch.cuda.synchronize()
        assert torch.equal(w, ref[0]) and torch.equal(m, ref[1]), t


def test_refusals():
    g = randn(8, 16)
    with pytest.raises(ValueError, match='float32, float16 or bfloat16'):
        optim.orthogonalize(g.double())
    with pytest.raises(ValueError, match='two dimensions'):
        optim.orthogonalize(g[0])
    with pytest.raises(ValueError, match='no backward'):
        optim.orthogonalize(g.clone().requires_grad_())
    with pytest.raises(ValueError, match='out must'):
        optim.orthogonalize(g, out=torch.empty(16, 8, device='cuda').t())
    with pytest.raises(_lib.MtazError, match='singular values grow'):
        optim.orthogonalize(g, steps=32, coefficients=(3.0, 0.0, 0.0))
    for bad in (0, 33):
        with pytest.raises(_lib.MtazError, match='steps'):
            optim.orthogonalize(g, steps=bad)
    m = torch.zeros_like(g)
    with pytest.raises(ValueError, match='twice'):
        optim.muon_step([g, g], [g, g], [m, m.clone()], lr=0.1)
    with pytest.raises(ValueError, match='momentum must be float32'):
        optim.muon_step([g], [g], [m.half()], lr=0.1)
    with pytest.raises(ValueError, match='contiguous'):
        optim.muon_step([g.t()], [g.t()], [m.t()], lr=0.1)
    with pytest.raises(_lib.MtazError, match='momentum'):
        optim.muon_step([g], [g], [m], lr=0.1, momentum=1.0)
    both = randn(2, 8, 16)
    flat = both.view(-1)
    with pytest.raises(ValueError, match='overlaps grad'):
        optim.orthogonalize(flat[:128].view(8, 16), out=flat[64:192].view(8, 16))
    with pytest.raises(ValueError, match='overlap'):
        optim.muon_step([flat[:128].view(8, 16), flat[64:192].view(8, 16)], [g, g], [m, m.clone()], lr=0.1)
    with pytest.raises(ValueError, match='a gradient overlaps'):
        optim.muon_step([g], [m], [m], lr=0.1)
    with pytest.raises(ValueError, match='a gradient overlaps'):
        optim.muon_step([both[0], both[1]], [both[1], g], [m, m.clone()], lr=0.1)


def test_shared_and_own_gradients():
    """One gradient for two parameters, and a gradient in its own parameter's place."""
    w, g = randn(2, 20, 60, seed=5), randn(20, 60, seed=6)
    m = torch.zeros(3, 20, 60, device='cuda')
    both = [w[0].clone(), w[1].clone()]
    optim.muon_step(both, [g, g], [m[0], m[1]], lr=0.1)
    for k in range(2):
        alone = w[k].clone()
        optim.muon_step([alone], [g], [torch.zeros_like(g)], lr=0.1)
        assert torch.equal(alone, both[k])
    own, want = w[0].clone(), w[0].clone()
    optim.muon_step([own], [own], [m[2]], lr=0.1)
    optim.muon_step([want], [w[0]], [torch.zeros_like(g)], lr=0.1)
    assert torch.equal(own, want)
