"""CPU: what records torch's operators sees the logits operators themselves (on tensors without data, as a tracer has
them), with the shapes, types and devices that they return."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from minitchess_alphazero_amd import logits as ops


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
