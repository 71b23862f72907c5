"""GPU: the learner operators where offsets pass 32 bits."""
import math

import pytest
import torch

from minitchess_alphazero_amd import logits as ops
from minitchess_alphazero_amd import optim

pytestmark = pytest.mark.gpu


def test_rows_behind_two_to_the_32():
    """4.36e9 logits: the first and last rows like the same rows alone."""
    rows, cols = 66000, 66001
    gen = torch.Generator(device='cuda').manual_seed(1)
    x = torch.empty(rows, cols, dtype=torch.float16, device='cuda').normal_(generator=gen)
    mask = torch.randint(-2 ** 31, 2 ** 31 - 1, (rows, (cols + 31) // 32), generator=gen, device='cuda').to(torch.int32)
    bias = torch.randn(cols, generator=gen, device='cuda')
    actions = torch.randint(0, cols, (rows, 5), generator=gen, device='cuda', dtype=torch.int32)
    ends = (slice(0, 2), slice(rows - 3, rows))
    y = ops.adjust_logits(x, mask, bias, actions, repetition=1.2, frequency=0.1, presence=0.2)
    for s in ends:
        assert torch.equal(y[s], ops.adjust_logits(x[s], mask[s], bias, actions[s], repetition=1.2, frequency=0.1, presence=0.2))
    target = y.zero_()                      # its room again: one target a row
    target.scatter_(1, actions[:, :1].long(), 1.0)
    loss, dz, _ = ops.policy_value_loss_grad(x, target, scale=float(rows))
    assert bool(loss.isfinite())
    for s in ends:
        n = s.stop - s.start
        assert torch.equal(dz[s], ops.policy_value_loss_grad(x[s].contiguous(), target[s].contiguous(), scale=float(n))[1])


@pytest.mark.parametrize('rows,cols', [(16384, 65536), (65536, 16384)])
def test_matrix_of_two_to_the_30(rows, cols):
    """Rows (columns) that are orthogonal and of one length: every singular value s is 1 / sqrt(r) of the norm, a step takes
    it to s (a + b s^2 + c s^4), and the result is the same entries times that."""
    r, long = min(rows, cols), max(rows, cols)
    at = torch.arange(r, device='cuda')
    other = (at * 4 + at % 3) % long        # distinct: 4 i, 4 i + 1, 4 i + 2
    g = torch.zeros(rows, cols, dtype=torch.bfloat16, device='cuda')
    places = (at, other) if rows == r else (other, at)
    g[places] = 0.5
    a, b, c = optim.COEFFICIENTS
    s = 1 / math.sqrt(r)
    for _ in range(5):
        s = s * (a + b * s ** 2 + c * s ** 4)
    got = optim.orthogonalize(g)
    # half a step of bfloat16, and what the tests of small matrices allow for five steps
    assert float((got[places].double() - s).abs().max()) <= (2.0 ** -8 + 2e-4) * abs(s)
    got[places] = 0
    assert not bool(got.any())
