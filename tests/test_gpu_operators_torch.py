"""GPU: the learner operators under what torch does with operators: tracing, streams, derivatives that they lack."""
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from minitchess_alphazero_amd import _lib
from minitchess_alphazero_amd import logits as ops
from minitchess_alphazero_amd import optim
from test_gpu_logits import gen, make, pack

pytestmark = pytest.mark.gpu


def inputs(seed, rows=6, cols=70):
    x, legal, actions, lengths = make(rows, cols, 9, seed)
    t = torch.rand(rows, cols, generator=gen(seed)) * legal
    v = torch.rand(rows, 1, generator=gen(seed + 1))
    return [a.cuda() for a in (x, torch.randn(cols, generator=gen(seed + 2)), v, pack(legal), actions, lengths, t)]


def step(x, b, v, mask, actions, lengths, t):
    """Adjusted logits into the loss, and back to logits, bias and value."""
    leaves = [a.detach().requires_grad_() for a in (x, b, v)]
    y = ops.adjust_logits(leaves[0], mask, leaves[1], actions, lengths, 1.2, 0.1, 0.3)
    loss = ops.policy_value_loss(y, t, leaves[2], torch.ones_like(v))
    return (y.detach(), loss.detach(), *torch.autograd.grad(loss, leaves), *ops.policy_value_loss_grad(x, t, legal=mask)[:2])


def test_traced_graph_computes():
    """The trace holds the operators, their backward passes too, and computes what the call does, for other inputs and on
    another stream than the one it was recorded on."""
    graph = make_fx(step)(*inputs(1))
    names = [str(n.target) for n in graph.graph.nodes if str(n.target).startswith('mtaz.')]
    assert sorted(set(names)) == ['mtaz.adjust_logits.default', 'mtaz.adjust_logits_back.default', 'mtaz.policy_loss.default',
                                  'mtaz.policy_loss_back.default', 'mtaz.policy_loss_grad.default']
    side = torch.cuda.Stream()
    for seed in (1, 2, 3):
        args = inputs(seed)
        want = step(*args)
        assert all(torch.equal(a, b) for a, b in zip(graph(*args), want))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = graph(*[a * 1 for a in args])   # a wrong stream would read these before they are there
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_tangents_are_refused_in_backward_too():
    x, b, v, mask, actions, lengths, t = inputs(4)
    y, loss = ops.adjust_logits(x.requires_grad_(), mask), ops.policy_value_loss(x, t)
    with forward_ad.dual_level():
        for out in (y, loss):
            g = torch.ones_like(out)
            with pytest.raises(ValueError, match='no forward-mode derivative'):
                torch.autograd.grad(out, x, forward_ad.make_dual(g, g), retain_graph=True)
        with pytest.raises(ValueError, match='no forward-mode derivative'):
            ops.adjust_logits(forward_ad.make_dual(x.detach(), x.detach()))
    torch.autograd.grad(loss, x)


def test_negated_views_are_the_numbers_they_show():
    """torch holds the imaginary part of a conjugate as a view that is negated when it is read."""
    def negated(*shape, seed):
        c = torch.randn(*shape, dtype=torch.complex64, generator=gen(seed)).cuda().conj()
        view = torch._neg_view(c.imag.neg().clone())      # contiguous, so that no copy resolves it on the way
        assert view.is_neg() and c.imag.is_neg() and torch.equal(view, c.imag)
        return view
    x, b = negated(6, 40, seed=1), negated(40, seed=2)
    t = torch.rand(6, 40, generator=gen(3)).cuda()
    plain = [a.clone() for a in (x, b)]
    want = ops.adjust_logits(plain[0], bias=plain[1])
    assert torch.equal(ops.adjust_logits(x, bias=b), want)
    assert torch.equal(ops.adjust_logits(x, bias=b, out=torch.empty_like(want)), want)
    for got, w in zip(ops.policy_value_loss_grad(x, t)[:2], ops.policy_value_loss_grad(plain[0], t)):
        assert torch.equal(got, w)
    assert torch.equal(optim.orthogonalize(x), optim.orthogonalize(plain[0]))
    ws, ms = [t.clone() for _ in range(2)], [torch.zeros_like(t) for _ in range(2)]
    optim.muon_step(ws, [x, plain[0]], ms, lr=0.1)
    assert torch.equal(ws[0], ws[1]) and torch.equal(ms[0], ms[1])
    with pytest.raises(ValueError, match='negated'):
        ops.adjust_logits(t, out=x)
    with pytest.raises(ValueError, match='negated'):
        optim.orthogonalize(t, out=x)
    for w, m in ((x, t), (t, x)):
        with pytest.raises(ValueError, match='negated'):
            optim.muon_step([w], [t.clone()], [m], lr=0.1)


@pytest.mark.parametrize('backend', ['eager', 'aot_eager'])
def test_compiled_functions_compute_the_same(backend):
    x, b, v, mask, actions, lengths, t = inputs(7)

    def loss(x, b):
        return ops.policy_value_loss(ops.adjust_logits(x, mask, b, actions, lengths, 1.2, 0.1, 0.3), t)
    both = []
    for f in (loss, torch.compile(loss, backend=backend)):
        leaves = [a.clone().requires_grad_() for a in (x, b)]
        out = f(*leaves)
        both.append((out, *torch.autograd.grad(out, leaves)))
    assert all(torch.equal(p, q) for p, q in zip(*both))


def test_operators_keep_what_their_schemas_say():
    """Schemas (nothing written, no aliases), registrations and the results without data, by torch's own checks."""
    x, b, v, mask, actions, lengths, t = inputs(9)
    nodes = _lib.nodes()
    leaf = [a.clone().requires_grad_() for a in (x, b, v)]
    for op, args in ((nodes.adjust_logits, (leaf[0], leaf[1], mask, actions, lengths, None, 1.2, 0.1, 0.2, True)),
                     (nodes.adjust_logits, (x, None, None, None, None, None, 1.0, 0.0, 0.0, False)),
                     (nodes.policy_loss, (leaf[0], leaf[2], t, torch.ones_like(v), mask)),
                     (nodes.policy_loss_grad, (x, v, t, torch.ones_like(v), mask, 2.0)),
                     (nodes.policy_loss_grad, (x, None, t, None, None, 1.0))):
        torch.library.opcheck(op.default, args)
