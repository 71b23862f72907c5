"""GPU: the policy/value loss in every form that a row's length selects, and outputs over their inputs.

Tolerances.  A term exp(z - top) of the softmax is off by |z - top| 2^-24 for the difference and as much for the factor
log2(e), and by 2 * 2^-24 for exp.  A row's sum has up to 64 own terms of a thread, 6 levels in a wave and 16 waves one
after the other; rows in tiles join these over up to 6 levels and as many steps as a lane has tiles (2 below), and each
join moves a sum by exp(-d) (off by (d + 2) 2^-24; all the d of a path together are at most the spread) and adds d pi to
the dot product: in all less than (4 spread + 160) 2^-24 of the sum of magnitudes.  A 16-bit gradient is rounded once."""
import ctypes
import math

import pytest
import torch

from minitchess_alphazero_amd import _lib
from minitchess_alphazero_amd import logits as ops
from test_gpu_logits import DTYPES, HALF, U, gen, loss64, make, pack

pytestmark = pytest.mark.gpu
TILE = 4096                                 # of float32 rows above 32768 columns; 8192 in 16 bits


def rows_of(cols, dtype, seed):
    """Six rows: ordinary, nothing legal, all at -inf, the first tiles masked, the top at the end, the first tiles at -inf."""
    z, legal, _, _ = make(6, cols, 1, seed, dtype, density=0.5)
    first = min(2 * TILE, cols // 2)
    z[2] = -math.inf
    legal[3, :first] = False
    z[3, :first] = math.nan
    z[4, -1], legal[4, -1] = 20.0, True
    z[5, :first] = -math.inf
    t = torch.rand(6, cols, generator=gen(seed + 1)) ** 3 * legal
    t = t / t.sum(1, keepdim=True).clamp(min=1e-6)
    t[2], t[5, :first] = 0.0, 0.0           # (with a target there the loss would be infinite)
    return z, legal, t


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('cols', [1024, 1025, 1100, 2048, 2049, 5000, 8192, 8193, 10007, 16384, 16385, 32768, 32769, 70001, 530001])
def test_loss_and_gradients(cols, dtype):
    z, legal, t = rows_of(cols, dtype, cols)
    for target_type in {torch.float32, dtype}:
        tt = t.to(target_type)
        want, g, size, spread, terms = loss64(z, tt, legal, None, None)
        tt = tt.masked_fill(~legal, math.nan)             # targets in masked places do not count
        cu = [a.cuda() for a in (z, tt, pack(legal))]
        loss, dz, _ = ops.policy_value_loss_grad(cu[0], cu[1], legal=cu[2])
        rel = (4 * spread + 160) * U
        assert abs(float(loss) - float(want)) <= rel * float(terms) + 4 * U * abs(float(want))
        tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
        assert bool(((dz.double().cpu() - g).abs() <= rel * size + HALF[dtype] * g.abs() + tiny).all())
        zl = cu[0].clone().requires_grad_()
        auto = ops.policy_value_loss(zl, cu[1], legal=cu[2])
        assert torch.equal(auto, loss)
        (3 * auto).backward()
        assert bool(((zl.grad.double().cpu() - 3 * g).abs() <= 3 * (rel * size + HALF[dtype] * g.abs()) + tiny).all())
        every, _, _, spread, terms = loss64(z[4:5], t[4:5].to(target_type), torch.ones(1, cols, dtype=torch.bool), None, None)
        got = ops.policy_value_loss(cu[0][4:5], t[4:5].to(target_type).cuda())   # without a mask
        assert abs(float(got) - float(every)) <= (4 * spread + 160) * U * float(terms) + 4 * U * abs(float(every))


@pytest.mark.parametrize('cols', [5000, 40000])
def test_values_and_rows_that_hold_no_number(cols):
    """A value term beside long rows; a target where the logit is -inf, and a NaN, stay in their row and gradient."""
    z, legal, t = rows_of(cols, torch.float32, 3)
    v, r = torch.rand(6, 1, generator=gen(1)), torch.ones(6, 1)
    want, g, *_ = loss64(z, t, legal, v, r)
    clean = ops.policy_value_loss_grad(*(a.cuda() for a in (z, t, v, r, pack(legal))))
    assert abs(float(clean[0]) - float(want)) <= 1e-5 * float(want)
    assert bool(((clean[2].double().cpu() - 2 * (v - r).double() / 6).abs() <= 6 * U).all())
    bad, tb = z.clone(), t.clone()
    bad[0, 7], legal[0, 7] = math.nan, True
    legal[5, 3], tb[5, 3] = True, 0.5
    loss, dz, dv = ops.policy_value_loss_grad(*(a.cuda() for a in (bad, tb, v, r, pack(legal))))
    assert bool(loss.isnan()) and bool(dz[0].isnan().any()) and torch.equal(dz[1:5], clean[1][1:5]) and torch.equal(dv, clean[2])
    bad[0, 7] = 0.0
    loss, dz, _ = ops.policy_value_loss_grad(*(a.cuda() for a in (bad, tb, v, r, pack(legal))))
    assert float(loss) == math.inf and bool(dz.isfinite().all())


def test_outputs_over_their_inputs():
    rows, cols = 5, 2100
    x, legal, actions, lengths = make(rows, cols, 4, 1)
    x, b, mask, actions, lengths = (a.cuda() for a in (x, torch.randn(rows, cols, generator=gen(2)), pack(legal), actions, lengths))
    want = ops.adjust_logits(x, mask, b, actions, lengths, 1.2, 0.1, 0.2)
    out = b.clone()
    assert torch.equal(ops.adjust_logits(x, mask, out, actions, lengths, 1.2, 0.1, 0.2, out=out), want)   # row over row
    with pytest.raises(_lib.MtazError, match='overlaps the mask, the bias'):
        ops.adjust_logits(x, bias=out[0], out=out)
    assert torch.equal(out, want)
    place = torch.zeros(rows * cols, dtype=torch.int32, device='cuda')
    words = place[:rows * mask.shape[1]].view(rows, -1)
    with pytest.raises(_lib.MtazError, match='overlaps the mask'):
        ops.adjust_logits(x, words, out=place.view(torch.float32).view(rows, cols))


def test_gradient_without_a_repetition_penalty_needs_no_logits():
    """Frequency and presence are constants: d x = d y where legal, also over the incoming gradient itself."""
    rows, cols = 3, 70
    _, legal, actions, _ = make(rows, cols, 6, 1, density=0.7)
    dy = torch.randn(rows, cols, generator=gen(1)).cuda()
    want = dy * legal.cuda()
    mask, actions = pack(legal).cuda(), actions.cuda()
    host = (ctypes.c_double * 3)(1.0, 0.25, 0.5)
    for dx in (torch.empty_like(dy), dy):
        _lib.check(_lib.lib().mtaz_adjust_logits_grad(
            0, rows, cols, 0, dy.data_ptr(), cols, None, 0, dx.data_ptr(), cols, None, 0, mask.data_ptr(), mask.stride(0),
            actions.data_ptr(), 6, 6, None, host, None, None, 0, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(dx, want)


@pytest.mark.parametrize('rows', [1, 15, 16, 17, 31, 32, 33])
def test_small_batches_captured_and_called(rows):
    """A captured call may take other launches than one that is made at once, and gives the same bits."""
    z, legal, _, _ = make(rows, 554, 1, rows, density=0.5)
    t = torch.rand(rows, 554, generator=gen(rows)) * legal
    v, r = torch.rand(rows, 1, generator=gen(1)), torch.ones(rows, 1)
    args = [a.cuda() for a in (z, t, v, r, pack(legal))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.policy_value_loss_grad(*args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.policy_value_loss_grad(*args)
    for k in range(4):
        args[0].mul_(0.75)
        graph.replay()
        want = ops.policy_value_loss_grad(*args)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        mean = loss64(args[0].cpu(), t, legal, v, r)[0]
        assert abs(float(want[0]) - float(mean)) <= 1e-5 * abs(float(mean))


@pytest.mark.parametrize('cols', [64, 2000, 20000, 40000])
def test_gradients_of_small_terms(cols):
    """float32 logits down to 80 below the top, which is 0, so that the differences are exact: each gradient k softmax is off
    by exp (2 U, and U for its correction), the sum of what is near the top (a handful of terms over up to 6 + 16 + 8
    additions, and 3 U of each), its reciprocal and four products, whatever its size: less than 45 U of itself."""
    z = torch.full((2, cols), -200.0)
    z[:, :64] = -torch.linspace(0, 80, 64)
    z[1] = z[1].flip(0)                     # the same from the last column on
    t = torch.zeros(2, cols)
    t[0, 0] = t[1, -1] = 1.0
    x = z.cuda().requires_grad_()
    ops.policy_value_loss(x, t.cuda()).backward()
    soft = z.double().softmax(1) / 2
    for dz in (ops.policy_value_loss_grad(z.cuda(), t.cuda())[1].cpu().double(), x.grad.cpu().double()):
        for row, there in ((0, slice(1, 64)), (1, slice(cols - 64, cols - 1))):
            assert float((dz[row, there] / soft[row, there] - 1).abs().max()) <= 45 * U
