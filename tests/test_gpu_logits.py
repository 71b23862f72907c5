"""GPU: adjust_logits, policy_value_loss and their gradients against the formulas in 64 bits.

Tolerances.  A 16-bit result is rounded once: half a step, eps / 2 of the value.  In float, an adjusted logit goes
through at most five operations: 5 * 2^-24 of the largest intermediate value.  A softmax term exp(z - top) is off by
|z - top| 2^-24 for the difference and 2 * 2^-24 for exp; a sum of n terms by at most log2-depth partial
sums: 16 own terms and 12 levels of joins, each 2^-24 relative to the sum of magnitudes."""
import math

import pytest
import torch

from minitchess_alphazero_amd import _lib
from minitchess_alphazero_amd import logits as ops

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -24
DTYPES = list(HALF)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def pack(legal):
    """Truth values [rows, cols] -> packed masks int32."""
    rows, cols = legal.shape
    words = (cols + 31) // 32
    bits = torch.zeros(rows, words * 32, dtype=torch.int64)
    bits[:, :cols] = legal.long()
    packed = (bits.view(rows, words, 32) << torch.arange(32)).sum(-1)
    return torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)


def make(rows, cols, history, seed, dtype=torch.float32, density=0.2):
    g = gen(seed)
    x = (3 * torch.randn(rows, cols, generator=g)).to(dtype)
    legal = torch.rand(rows, cols, generator=g) < density
    if rows > 2:
        legal[1] = False
    actions = torch.randint(-2, cols + 2, (rows, history), generator=g, dtype=torch.int32)
    if history > 2:
        actions[:, 1] = actions[:, 0]
    lengths = torch.randint(0, history + 1, (rows,), generator=g, dtype=torch.int32)
    return x, legal, actions, lengths


def counts(actions, lengths, cols):
    c = torch.zeros(actions.shape[0], cols, dtype=torch.float64)
    for r in range(actions.shape[0]):
        a = actions[r, :max(0, int(lengths[r])) if lengths is not None else None].long()
        a = a[(a >= 0) & (a < cols)]
        c[r] = torch.bincount(a, minlength=cols)[:cols].double()
    return c


def adjusted(x, legal, bias, c, rep, freq, pres):
    """64 bits: (y before the mask, its slope, the largest intermediate magnitude)"""
    x = x.double()
    rep, freq, pres = (torch.as_tensor(t, dtype=torch.float64).reshape(-1, 1) for t in (rep, freq, pres))
    slope = torch.where(c > 0, torch.where(x > 0, 1 / rep, rep.expand_as(x)), torch.ones_like(x))
    y = x * slope - c * freq - (c > 0) * pres
    size = (x * slope).abs() + (c * freq).abs() + pres.abs()
    if bias is not None:
        y = y + bias.double()
        size = size + bias.double().abs()
    return y, slope, size


SHAPES = [(1, 1, 1), (3, 5, 2), (4, 554, 60), (2, 4095, 9), (2, 4097, 300), (1, 20011, 1000), (5, 33, 0)]


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('rows,cols,history', SHAPES)
def test_adjust(rows, cols, history, dtype):
    x, legal, actions, lengths = make(rows, cols, history, rows + cols, dtype)
    g = gen(1)
    for masks in (None, legal, legal[:1]):
        for bias in (None, torch.randn(cols, generator=g), torch.randn(rows, cols, generator=g)):
            pen = (1.3, 0.25, 0.5)
            c = counts(actions, lengths, cols)
            y, _, size = adjusted(x, legal, bias, c, *pen)
            got = ops.adjust_logits(x.cuda(), None if masks is None else pack(masks).cuda(),
                                    None if bias is None else bias.cuda(), actions.cuda() if history else None,
                                    lengths.cuda() if history else None, *pen).cpu()
            keep = torch.ones_like(x, dtype=torch.bool) if masks is None else masks.expand(rows, cols)
            assert got.dtype == dtype and bool((got[~keep] == -math.inf).all())
            err = (got.double() - y).abs()[keep]
            assert bool((err <= (5 * U * size + HALF[dtype] * y.abs() + 1e-12 + (2.0 ** -25 if dtype == torch.float16 else 0))[keep]).all())


def test_adjust_per_row_penalties_and_lengths():
    rows, cols = 6, 777
    x, legal, actions, _ = make(rows, cols, 40, 5)
    lengths = torch.tensor([0, 1, 40, 99, -5, 7], dtype=torch.int32)   # beyond the list and below 0 are cut
    rep, freq, pres = 0.5 + torch.rand(rows), torch.randn(rows), torch.randn(rows)
    c = counts(actions, lengths.clamp(0, 40), cols)
    y, _, size = adjusted(x, legal, None, c, rep, freq, pres)
    got = ops.adjust_logits(x.cuda(), None, None, actions.cuda(), lengths.cuda(), rep.cuda(), freq.cuda(), pres.cuda())
    assert bool(((got.double().cpu() - y).abs() <= 5 * U * size).all())
    c = counts(actions, None, cols)
    y, _, size = adjusted(x, legal, None, c, rep, 0.5, pres)
    got = ops.adjust_logits(x.cuda(), actions=actions.cuda(), repetition=rep.cuda(), frequency=0.5, presence=pres.cuda())
    assert bool(((got.double().cpu() - y).abs() <= 5 * U * size).all())


def test_adjust_layouts_in_place_and_poison():
    """Row strides, views that start at odd elements, in place; NaN and infinities in masked places stay there;
    what lies between and behind the rows of out is not written."""
    rows, cols = 7, 261
    x, legal, actions, lengths = make(rows, cols, 12, 8, torch.bfloat16)
    x[~legal] = torch.tensor([math.nan, math.inf, -math.inf])[torch.arange(int((~legal).sum())) % 3].bfloat16()
    args = (pack(legal).cuda(), None, actions.cuda(), lengths.cuda(), 1.2, 0.1, 0.2)
    want = ops.adjust_logits(x.cuda(), *args)
    assert not want.isnan().any() and bool((want == -math.inf).cpu().eq(~legal).all())
    wide = torch.full((rows + 1, 300), 7.0, dtype=torch.bfloat16, device='cuda')
    view = wide[:rows, 5:5 + cols]
    view.copy_(x.cuda())
    out = torch.full((rows + 1, 301), 9.0, dtype=torch.bfloat16, device='cuda')
    ops.adjust_logits(view, *args, out=out[:rows, 3:3 + cols])
    assert torch.equal(out[:rows, 3:3 + cols], want)
    assert bool((out[:, :3] == 9).all()) and bool((out[:, 3 + cols:] == 9).all()) and bool((out[rows] == 9).all())
    assert ops.adjust_logits(view, *args, out=view) is view
    assert torch.equal(view, want) and bool((wide[:, 5 + cols:] == 7).all()) and bool((wide[rows] == 7).all())
    assert torch.equal(ops.adjust_logits(x.cuda().t().contiguous().t(), *args), want)
    assert ops.adjust_logits(x.cuda()[:0]).shape == (0, cols)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('rows,cols,history', [(1, 1, 1), (4, 554, 60), (130, 97, 5), (3, 4099, 64)])
def test_adjust_backward(rows, cols, history, dtype):
    x, legal, actions, lengths = make(rows, cols, history, 3 * rows + cols, dtype)
    dy = torch.randn(rows, cols, generator=gen(9)).to(dtype)
    dy[~legal] = math.nan                   # must not come through the mask
    c = counts(actions, lengths, cols)
    _, slope, _ = adjusted(x, legal, None, c, 1.4, 0.1, 0.2)
    g64 = torch.where(legal, dy.double(), 0.0)
    for shape in (None, (cols,), (1, cols), (rows, cols)):
        z = x.cuda().requires_grad_()
        b = None if shape is None else torch.zeros(shape, device='cuda', requires_grad=True)
        y = ops.adjust_logits(z, pack(legal).cuda(), b, actions.cuda(), lengths.cuda(), 1.4, 0.1, 0.2)
        y.backward(dy.cuda())
        want = g64 * slope
        assert bool(((z.grad.double().cpu() - want).abs() <= (HALF[dtype] + 3 * U) * want.abs() + 2.0 ** -25 * (dtype == torch.float16)).all())
        if b is not None:
            wb = g64 if b.dim() == 2 and b.shape[0] == rows else g64.sum(0).view(shape)
            size = (g64 if b.dim() == 2 and b.shape[0] == rows else g64).abs().sum(0)
            assert b.grad.shape == b.shape and bool(((b.grad.double().cpu() - wb).abs() <= (rows + 64) * U * size).all())


@pytest.mark.parametrize('rows,cols', [(3000, 61), (1500, 1300), (17, 5000)])
def test_adjust_backward_many_rows(rows, cols):
    """Several rows a workgroup, without and with a bias they share, and gradients that are broadcast views."""
    x, legal, _, _ = make(rows, cols, 1, rows, density=0.5)
    mask = pack(legal).cuda()
    for dy in (torch.randn(rows, cols, generator=gen(3)), torch.randn(1, cols, generator=gen(4)).expand(rows, cols),
               torch.ones(1, 1).expand(rows, cols)):
        for shape in ((cols,), (rows, cols)):
            z, b = x.cuda().requires_grad_(), torch.zeros(shape, device='cuda', requires_grad=True)
            ops.adjust_logits(z, mask, b).backward(dy.cuda() if dy.stride(0) else dy[:1].cuda().expand(rows, cols))
            want = torch.where(legal, dy, 0.0)
            assert torch.equal(z.grad.cpu(), want)
            if b.dim() == 2:
                assert torch.equal(b.grad.cpu(), want)
            else:
                size = want.double().abs().sum(0)
                assert bool(((b.grad.double().cpu() - want.double().sum(0)).abs() <= (rows + 64) * U * size).all())


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_adjust_many_rows_share_bias_and_mask(dtype):
    rows, cols = 4097, 1100                 # an odd number of rows, two a workgroup
    x, legal, actions, lengths = make(rows, cols, 20, 6, dtype)
    bias = torch.randn(cols, generator=gen(2))
    got = ops.adjust_logits(x.cuda(), pack(legal[:1]).cuda(), bias.cuda(), actions.cuda(), lengths.cuda(), 1.3, 0.25, 0.5).cpu()
    y, _, size = adjusted(x, legal[:1], bias, counts(actions, lengths, cols), 1.3, 0.25, 0.5)
    keep = legal[:1].expand(rows, cols)
    assert bool((got[~keep] == -math.inf).all())
    err = (got.double() - y).abs()[keep]
    assert bool((err <= (5 * U * size + HALF[dtype] * y.abs() + 1e-12 + (2.0 ** -25 if dtype == torch.float16 else 0))[keep]).all())


def test_columns_of_one_matrix_and_overlaps():
    both = torch.randn(6, 80, generator=gen(1)).cuda()
    want = ops.adjust_logits(both[:, :40], bias=both.new_ones(40))
    ops.adjust_logits(both[:, :40], bias=both.new_ones(40), out=both[:, 40:])
    assert torch.equal(both[:, 40:], want)
    with pytest.raises(_lib.MtazError, match='overlaps'):
        ops.adjust_logits(both[:, :40], out=both[:, 39:79])
    with pytest.raises(_lib.MtazError, match='overlaps'):
        ops.adjust_logits(both[:5], out=both[1:])


def test_adjust_gradient_against_differences():
    x, legal, actions, lengths = make(3, 40, 10, 2, density=0.6)
    x = x + 0.5 * x.sign()                  # no logit within a step of 0, where the slope jumps
    w = torch.randn(3, 40, generator=gen(4))
    w[~legal] = 0
    z = x.cuda().requires_grad_()
    args = (pack(legal).cuda(), None, actions.cuda(), lengths.cuda(), 1.4, 0.1, 0.2)

    def value(t):
        y = ops.adjust_logits(t, *args)
        return (torch.where(y == -math.inf, 0.0, y).double() * w.cuda().double()).sum()
    value(z).backward()
    h = 2.0 ** -5
    for r, v in ((0, 3), (0, 17), (2, 5), (2, 39)):
        d = torch.zeros_like(x)
        d[r, v] = h
        with torch.no_grad():
            slope = float(value((x + d).cuda()) - value((x - d).cuda())) / (2 * h)
        # linear between the two points: the difference carries the roundings of its two values, 5 * 2^-24 of |x| <= 20 each
        assert abs(slope - float(z.grad[r, v])) <= 2 * 5 * U * 20 * abs(float(w[r, v])) / (2 * h) + 4 * U * abs(slope)


def test_adjust_bias_gradient_is_repeatable():
    rows, cols = 300, 1001
    dy = torch.randn(rows, cols, generator=gen(1)).cuda()
    x = torch.randn(rows, cols, generator=gen(2)).cuda()

    def grads():
        b = torch.zeros(cols, device='cuda', requires_grad=True)
        ops.adjust_logits(x, bias=b).backward(dy)
        return b.grad
    first = grads()
    assert all(torch.equal(grads(), first) for _ in range(3))


def loss64(z, t, legal, v, r):
    z, t = z.double(), t.double()
    z = z.masked_fill(~legal, -math.inf)
    t = t.masked_fill(~legal, 0.0)
    some = (z > -math.inf).any(1)
    lse = torch.where(some, torch.logsumexp(z, 1), torch.zeros(len(z), dtype=torch.float64))
    terms = torch.where(t != 0, t * (lse[:, None] - z), 0.0)
    row = torch.where(some, terms.sum(1), 0.0)
    soft = torch.where(z > -math.inf, (z - lse[:, None]).exp(), 0.0)
    g = torch.where(some[:, None] & legal, soft * t.sum(1, keepdim=True) - t, 0.0)
    size = soft * t.abs().sum(1, keepdim=True) + t.abs()
    spread = (z - z.max(1, keepdim=True).values).masked_fill(z == -math.inf, 0.0).abs().max()
    if v is not None:
        row = row + (v.double() - r.double()).view(-1) ** 2
    return row.mean(), g / len(z), size / len(z), float(spread.nan_to_num(0.0)), terms.abs().sum(1).mean()


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('rows,cols', [(1, 1), (2, 3), (32, 554), (300, 61), (3, 4096), (2, 4097), (2, 30011)])
def test_loss_and_gradients(rows, cols, dtype):
    z, legal, _, _ = make(rows, cols, 1, rows * cols, dtype, density=0.5)
    if rows > 2:
        z[2] = -math.inf                    # legal, but out of the question
    for target_type in {torch.float32, dtype}:
        for masks, value in ((legal, True), (legal, False), (None, True)):
            t = torch.rand(rows, cols, generator=gen(3)) ** 3
            if masks is not None:
                t = t * masks
            t = t / t.sum(1, keepdim=True).clamp(min=1e-6)
            if masks is not None:
                t[~masks] = math.nan        # targets in masked places do not count
            t = t.to(target_type)
            if rows > 2:
                t[2] = 0                    # (with a target there the loss would be infinite)
            v, r = (torch.tanh(torch.randn(rows, 1, generator=gen(4))), torch.sign(torch.randn(rows, 1, generator=gen(5)))) if value else (None, None)
            every = torch.ones(rows, cols, dtype=torch.bool) if masks is None else masks
            want, g, size, spread, terms = loss64(z, t.masked_fill(~every, 0.0), every, v, r)
            cu = [None if a is None else a.cuda() for a in (t, v, r, None if masks is None else pack(masks))]
            loss, dz, dv = ops.policy_value_loss_grad(z.cuda(), *cu)
            # each term: difference, exp and the 28 partial sums
            rel = (2 * spread + 40) * U
            assert abs(float(loss) - float(want)) <= rel * (float(terms) + 3.0) + 4 * U * abs(float(want))
            tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
            assert bool(((dz.double().cpu() - g).abs() <= rel * size + HALF[dtype] * g.abs() + tiny).all())
            zl = z.cuda().requires_grad_()
            vl = None if v is None else v.cuda().requires_grad_()
            auto = ops.policy_value_loss(zl, cu[0], vl, cu[2], cu[3])
            assert torch.equal(auto, loss)
            (3 * auto).backward()
            assert bool(((zl.grad.double().cpu() - 3 * g).abs() <= 3 * (rel * size + HALF[dtype] * g.abs()) + tiny).all())
            if value:
                dv64 = 2 * (v.double() - r.double()) / rows
                assert bool(((dv.double().cpu() - dv64).abs() <= 6 * U * dv64.abs() + 1e-12).all())
                assert vl.grad.shape == v.shape and bool(((vl.grad.double().cpu() - 3 * dv64).abs() <= 18 * U * dv64.abs() + 1e-12).all())


def test_loss_extremes():
    z = torch.tensor([[1e30, -1e30, 0.0], [1e4, 1e4 - 1, 0.0], [math.nan, 0.0, 1.0], [-math.inf, 1.0, 2.0], [0.0, 0.0, 0.0]])
    t = torch.tensor([[1.0, 0.0, 0.0], [0.5, 0.5, 0.0], [1.0, 0.0, 0.0], [0.0, 0.5, 0.5], [0.25, 0.5, 0.0]])
    legal = torch.ones(5, 3, dtype=torch.bool)
    legal[2, 0] = False
    want, g, *_ = loss64(z, t, legal, None, None)
    loss, dz, dv = ops.policy_value_loss_grad(z.cuda(), t.cuda(), legal=pack(legal).cuda())
    assert dv is None
    assert abs(float(loss) - float(want)) <= 1e-6 and float((dz.double().cpu() - g).abs().max()) <= 1e-6
    one, dz, _ = ops.policy_value_loss_grad(z[3:4].cuda(), torch.tensor([[0.5, 0.5, 0.0]]).cuda())
    assert float(one) == math.inf           # a target where the logit is -inf
    assert bool(ops.policy_value_loss_grad(z[2:3].cuda(), t[2:3].cuda())[0].isnan())
    only = torch.tensor([[math.nan, 0.0, 0.0]])
    assert bool(ops.policy_value_loss_grad(only.cuda(), t[:1].cuda(), legal=pack(torch.tensor([[True, False, False]])).cuda())[0].isnan())
    huge = 300.0 * torch.randn(2, 9, generator=gen(1)) ** 3   # one-hot softmax, far apart
    tt = torch.full((2, 9), 1 / 9)
    want, g, _, spread, terms = loss64(huge, tt, torch.ones(2, 9, dtype=torch.bool), None, None)
    loss, dz, _ = ops.policy_value_loss_grad(huge.cuda(), tt.cuda())
    assert abs(float(loss) - float(want)) <= 40 * U * float(terms) + 1e-6


def test_loss_gradient_against_differences():
    z, legal, _, _ = make(4, 30, 1, 6, density=0.7)
    t = torch.rand(4, 30, generator=gen(7)) * legal
    v, r = torch.rand(4, generator=gen(8)), torch.ones(4)
    args = [a.cuda() for a in (t, v, r, pack(legal))]
    _, dz, dv = ops.policy_value_loss_grad(z.cuda(), *args)
    h = 2.0 ** -4
    for b, a in ((0, 0), (2, 11), (3, 29)):
        d = torch.zeros_like(z)
        d[b, a] = h
        up, down = (float(ops.policy_value_loss((z + s * d).cuda(), *args)) for s in (1, -1))
        # third derivative of the loss in one logit: at most sum of targets / rows * 0.1; and two roundings of the loss
        bound = float(t[b].sum()) / 4 * 0.1 * h * h / 6 + 60 * U * max(abs(up), 1.0) / h
        assert abs((up - down) / (2 * h) - float(dz[b, a])) <= bound


def test_adjusted_logits_into_the_loss_captured():
    """Adjusted logits need no mask in the loss: the same loss and gradients; the whole chain captured, replayed with
    eager work between, against the eager chain."""
    rows, cols = 9, 554
    x, legal, actions, lengths = make(rows, cols, 30, 11)
    t = torch.rand(rows, cols, generator=gen(12)) * legal
    v, r = torch.rand(rows, 1, generator=gen(13)).cuda(), torch.ones(rows, 1, device='cuda')
    x, t, actions, lengths, mask = (a.cuda() for a in (x, t, actions, lengths, pack(legal)))

    def chain(z, b, val):
        y = ops.adjust_logits(z, mask, b, actions, lengths, 1.2, 0.1, 0.3)
        loss = ops.policy_value_loss(y, t, val, r)
        return (loss, *torch.autograd.grad(loss, (z, b, val)))

    leaves = [a.detach().requires_grad_() for a in (x, torch.zeros(cols, device='cuda'), v)]
    eager = chain(*leaves)
    masked = ops.policy_value_loss(ops.adjust_logits(x, None, None, actions, lengths, 1.2, 0.1, 0.3), t, v, r, mask)
    assert torch.equal(masked, eager[0])
    static = [a.detach().clone().requires_grad_() for a in leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(*static)
    for k in range(3):
        with torch.no_grad():
            for a in static:
                a.add_(0.125)
        graph.replay()
        want = chain(*[a.detach().clone().requires_grad_() for a in static])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_legal_masks_and_positions():
    import numpy as np
    from minitchess_alphazero_amd.environment import pos_from_fen, pos_legal
    from conftest import LONG_LIST_FENS
    fens = ['2nbk/2ppp/5/5/PPP2/KBN2 w 0 1', 'k4/2K2/5/5/5/1Q3 b 0 5'] + LONG_LIST_FENS
    pos = np.stack([pos_from_fen(f) for f in fens])
    masks = ops.legal_masks(pos, 'cuda').cpu()
    for m, p in zip(masks, pos):
        want = torch.zeros(1, 554, dtype=torch.bool)
        want[0, pos_legal(p)] = True
        assert torch.equal(pack(want)[0], m)


def test_refusals():
    x = torch.zeros(3, 40, device='cuda')
    i32 = dict(dtype=torch.int32, device='cuda')
    with pytest.raises(ValueError, match='rows, cols'):
        ops.adjust_logits(x[0])
    with pytest.raises(ValueError, match='float32, float16 or bfloat16'):
        ops.adjust_logits(x.double())
    with pytest.raises(ValueError, match='legal has shape'):
        ops.adjust_logits(x, legal=torch.zeros(3, 1, **i32))
    with pytest.raises(ValueError, match='legal must be torch.int32'):
        ops.adjust_logits(x, legal=torch.zeros(3, 2, dtype=torch.int64, device='cuda'))
    with pytest.raises(ValueError, match='bias'):
        ops.adjust_logits(x, bias=torch.zeros(40, dtype=torch.bfloat16, device='cuda'))
    with pytest.raises(ValueError, match='actions must be'):
        ops.adjust_logits(x, actions=torch.zeros(3, 5, dtype=torch.int64, device='cuda'))
    with pytest.raises(ValueError, match='lengths without'):
        ops.adjust_logits(x, lengths=torch.zeros(3, **i32))
    for bad in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match='positive'):
            ops.adjust_logits(x, actions=torch.zeros(3, 5, **i32), repetition=bad)
    with pytest.raises(ValueError, match='out is not supported'):
        ops.adjust_logits(x.clone().requires_grad_(), out=torch.empty_like(x))
    with pytest.raises(ValueError, match='do not overlap'):
        ops.adjust_logits(x, out=torch.empty(1, 40, device='cuda').expand(3, 40))
    with pytest.raises(ValueError, match='no rows'):
        ops.policy_value_loss(x[:0], x[:0])
    with pytest.raises(ValueError, match='come together'):
        ops.policy_value_loss(x, x, value=torch.zeros(3, device='cuda'))
    with pytest.raises(ValueError, match='value must be'):
        ops.policy_value_loss(x, x, torch.zeros(3, device='cuda').half(), torch.zeros(3, device='cuda'))
    with pytest.raises(ValueError, match='target has shape'):
        ops.policy_value_loss(x, x[:, :39])
    with pytest.raises(ValueError, match='have no gradient'):
        ops.policy_value_loss(x, x.clone().requires_grad_())
    y = x.clone().requires_grad_()
    loss = ops.policy_value_loss(y, torch.softmax(x, 1))
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()
    assert _lib.lib().mtaz_policy_loss_workspace(-1, 5) < 0


def test_gradients_are_not_differentiated_again():
    x = torch.randn(3, 40, generator=gen(1)).cuda().requires_grad_()
    b = torch.zeros(40, device='cuda', requires_grad=True)
    t = torch.softmax(x.detach(), 1)
    for y in (ops.adjust_logits(x, bias=b).square().sum(), ops.policy_value_loss(x + b, t)):
        dx, db = torch.autograd.grad(y, (x, b), create_graph=True)
        with pytest.raises(RuntimeError, match='twice'):
            (dx.sum() + db.sum()).backward()
    only = torch.autograd.grad(ops.adjust_logits(x.detach(), bias=b).sum(), b)[0]     # one of the two wanted
    assert torch.equal(only, torch.full_like(b, 3.0))
    v = torch.ones(3, 1, device='cuda', requires_grad=True)
    dv, = torch.autograd.grad(ops.policy_value_loss(x.detach(), t, v, torch.zeros_like(v)), v)
    assert bool(((dv - 2 / 3).abs() <= 4 * U).all())
    assert not ops.policy_value_loss(x.detach(), t).requires_grad
    with torch.no_grad():
        assert not ops.policy_value_loss(x, t).requires_grad and not ops.adjust_logits(x).requires_grad
