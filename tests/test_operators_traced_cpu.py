"""CPU: what records torch's operators sees the logits operators themselves (on tensors without data, as a tracer has
them), with the shapes, types and devices that they return."""
import pytest
import torch
from torch.autograd import forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from minitchess_alphazero_amd import logits as ops
from minitchess_alphazero_amd import optim


def called(graph):
    return [str(n.target) for n in graph.graph.nodes if n.op == 'call_function' and str(n.target).startswith('mtaz.')]


@pytest.fixture
def fake():
    with FakeTensorMode():
        yield


def tensors(rows, cols, dtype=torch.bfloat16):
    on = dict(device='cuda')
    return (torch.empty(rows, cols, dtype=dtype, **on), torch.empty(rows, cols, **on), torch.empty(rows, 1, **on),
            torch.empty(rows, (cols + 31) // 32, dtype=torch.int32, **on), torch.empty(rows, 7, dtype=torch.int32, **on))


def test_operators_stay_in_the_graph(fake):
    z, t, v, mask, actions = tensors(5, 40)
    graph = make_fx(lambda z, m, a: ops.adjust_logits(z, m, actions=a, repetition=1.2))(z, mask, actions)
    assert called(graph) == ['mtaz.adjust_logits.default']
    graph = make_fx(lambda z, t, v, m: ops.policy_value_loss(z, t, v, v, m))(z, t, v, mask)
    assert called(graph) == ['mtaz.policy_loss.default']
    graph = make_fx(lambda z, t, v, m: ops.policy_value_loss_grad(z, t, v, v, m, 2.0))(z, t, v, mask)
    assert called(graph) == ['mtaz.policy_loss_grad.default']


def test_shapes_without_data(fake):
    z, t, v, mask, actions = tensors(5, 40)
    y = ops.adjust_logits(z.t().contiguous().t(), mask, torch.empty(40, device='cuda'), actions)
    assert (y.shape, y.dtype, y.device, y.is_contiguous()) == ((5, 40), torch.bfloat16, z.device, True)
    loss = ops.policy_value_loss(z, t, v, v, mask)
    assert (loss.shape, loss.dtype, loss.device) == ((), torch.float32, z.device)
    loss, dz, dv = ops.policy_value_loss_grad(z, t, v, v)
    assert (loss.shape, dz.shape, dz.dtype, dv.shape, dv.dtype) == ((), (5, 40), torch.bfloat16, (5, 1), torch.float32)
    assert ops.policy_value_loss_grad(z, t)[2] is None


def test_tangents_are_refused(fake):
    """No operator has a forward-mode derivative: a result without a tangent would say that it is 0."""
    z, t, v, mask, actions = tensors(5, 40, torch.float32)
    per_row = torch.ones(5, device='cuda')
    with forward_ad.dual_level():
        d, dv, dp = (forward_ad.make_dual(a, torch.ones_like(a)) for a in (z, v, per_row))
        for call in (lambda: ops.adjust_logits(d), lambda: ops.adjust_logits(z, bias=forward_ad.make_dual(z[0].clone(), z[1])),
                     lambda: ops.adjust_logits(z, actions=actions, repetition=dp), lambda: ops.adjust_logits(d, out=z),
                     lambda: ops.adjust_logits(z, out=d), lambda: ops.policy_value_loss(d, t),
                     lambda: ops.policy_value_loss(z, t, dv, v), lambda: ops.policy_value_loss(z, t, v, dv),
                     lambda: ops.policy_value_loss(z, d), lambda: ops.policy_value_loss_grad(d, t),
                     lambda: optim.orthogonalize(d), lambda: optim.orthogonalize(z, out=d),
                     lambda: optim.muon_step([d], [z], [t], lr=0.1), lambda: optim.muon_step([z], [d], [t], lr=0.1),
                     lambda: optim.muon_step([z], [t], [d], lr=0.1)):
            with pytest.raises(ValueError, match='no forward-mode derivative'):
                call()
        for call in (lambda: ops.adjust_logits(d.clone().requires_grad_()), lambda: ops.policy_value_loss(d.clone().requires_grad_(), t)):
            with pytest.raises(ValueError, match='no forward-mode derivative'):
                call()
        assert ops.policy_value_loss(z, t).shape == ()
    assert ops.adjust_logits(z).shape == (5, 40)


def test_calls_that_a_tracer_would_lose_are_refused(fake):
    z, t, v, mask, actions = tensors(5, 40, torch.float32)
    pos = torch.zeros(5, 5, dtype=torch.int32, device='cuda')

    def step(z):
        optim.muon_step([z], [t], [t.clone()], lr=0.1)
        return z
    for call in (lambda z: optim.orthogonalize(z), step, lambda z: ops.adjust_logits(z, out=z), lambda z: ops.legal_masks(pos, 'cuda')):
        with pytest.raises(RuntimeError, match='cannot be traced'):
            make_fx(call)(z)
