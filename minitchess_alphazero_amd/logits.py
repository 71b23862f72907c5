"""Operators on action logits [rows, cols], on hand-written HIP kernels (csrc/mtaz_logits.hip).

    adjust_logits           penalties for repeated actions, a bias and a legal-move mask; differentiable
    policy_value_loss       the learner's loss (exp/learner.py:86-87) over the legal moves; differentiable
    policy_value_loss_grad  that loss and its gradients in one call
    legal_masks             the packed legal masks of positions (mtaz_legal_batch)

A mask is packed 32 actions a word: action v is legal where bit v & 31 of word v >> 5 is set, int32
[rows, ceil(cols / 32)], or [1, words] / [words] for one mask that all rows share.  Logits are float32,
float16 or bfloat16, sums are float32, and the operators enqueue on the current stream without a
synchronization; they may be captured in a HIP graph (a backward pass like any of torch's: with no eager graph of the
same leaves alive).  There is no CPU form: tensors elsewhere are refused, and so are tensors that carry a tangent of
forward-mode differentiation.
"""
import torch

from . import _lib
from .environment import MOVE_CAP, RULES_FLAGS
from .optim import TYPES, _check_type, _doubles, _no_tangent, _not_traced, _stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _unit(t):
    """t with its last dimension dense (a copy where it is not)."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _row_stride(t):
    """Elements from one row to the next; 0 where one row serves all."""
    return 0 if t is None or t.dim() == 1 or t.shape[0] == 1 else t.stride(0)


def _check_rows(t, what, like, shapes, dtypes):
    if t.device != like.device:
        raise ValueError(f'{what} must be on {like.device}, not on {t.device}')
    if t.dtype not in dtypes:
        raise ValueError(f'{what} must be {" or ".join(str(d) for d in dtypes)}, not {t.dtype}')
    if t.shape not in shapes:
        raise ValueError(f'{what} has shape {tuple(t.shape)}, expected {" or ".join(str(s) for s in shapes)}')


def _call(op, *args):
    try:
        return op(*args)
    except RuntimeError as e:
        text = str(e)
        if not text.startswith('mtaz error '):
            raise
        code, why = text[len('mtaz error '):].split(': ', 1)
        raise _lib.MtazError(int(code), why) from None


def _check_logits(logits):
    _check_type(logits, 'logits')
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f'logits must be [rows, cols], got {tuple(logits.shape)}')


def _check_legal(legal, logits):
    if legal is not None:
        rows, words = logits.shape[0], (logits.shape[1] + 31) // 32
        _check_rows(legal, 'legal', logits, ((rows, words), (1, words), (words,)), (torch.int32, torch.uint32))


def legal_masks(positions, device, rules_flags=RULES_FLAGS, move_cap=MOVE_CAP):
    """Packed legal masks [n, 18] int32 of packed positions [n, 5] (host uint32 or device int32): what
    mtaz_legal_batch finds (it waits for the stream, unlike the other functions here).  A position with no
    legal move has an empty mask."""
    import numpy as np
    _not_traced('legal_masks')
    dev = torch.device(device)
    if not torch.is_tensor(positions):
        positions = torch.from_numpy(np.ascontiguousarray(positions, np.uint32).view(np.int32)).to(dev)
    if positions.dim() != 2 or positions.shape[1] != 5 or positions.dtype != torch.int32 or positions.device.type != 'cuda':
        raise ValueError('positions must be [n, 5] 32-bit words')
    pos = positions.contiguous()
    n = pos.shape[0]
    codes = torch.empty((n, _lib.KMAX), dtype=torch.int16, device=pos.device)
    counts, outcomes = (torch.empty(n, dtype=torch.int32, device=pos.device) for _ in range(2))
    masks = torch.zeros((n, 18), dtype=torch.int32, device=pos.device)
    if n:
        _lib.check(_lib.lib().mtaz_legal_batch(pos.device.index, pos.data_ptr(), n, rules_flags, move_cap, codes.data_ptr(),
                                               counts.data_ptr(), masks.data_ptr(), outcomes.data_ptr(),
                                               _stream(pos.device)))
    return masks


# ---- penalties, bias and mask ----------------------------------------------------------------------------
class _Taken:
    """The actions taken and their penalties: tensors = (actions, lengths, penalties per row), host = the penalties that
    are numbers, bends = whether the slope is other than 1 somewhere."""
    __slots__ = ('tensors', 'host', 'bends')

    def __init__(self, logits, actions, lengths, repetition, frequency, presence):
        rows = logits.shape[0]
        given = (repetition, frequency, presence)
        tensors = [t for t in given if isinstance(t, torch.Tensor)]
        for t in tensors:
            _check_rows(t, 'a penalty', logits, ((rows,),), (torch.float32,))
            if t.requires_grad and torch.is_grad_enabled():
                raise ValueError('penalties have no gradient')
        per_row_repetition = isinstance(repetition, torch.Tensor)
        if not per_row_repetition and not repetition > 0:
            raise ValueError(f'repetition must be positive, got {repetition}')
        self.host = (1.0, 0.0, 0.0) if tensors else (float(repetition), float(frequency), float(presence))
        if actions is None:
            if lengths is not None:
                raise ValueError('lengths without actions')
            self.tensors, self.bends = (None, None, None), False
            return
        if actions.dim() != 2:
            raise ValueError(f'actions must be [rows, history], got {tuple(actions.shape)}')
        _check_rows(actions, 'actions', logits, ((rows, actions.shape[1]),), (torch.int32,))
        if actions.shape[1] > 1 << 30:
            raise ValueError(f'actions hold at most 2^30 entries a row, got {actions.shape[1]}')
        if lengths is not None:
            _check_rows(lengths, 'lengths', logits, ((rows,),), (torch.int32,))
            lengths = lengths.contiguous()
        actions = _unit(actions)
        per_row = None
        if tensors:
            like = dict(dtype=torch.float32, device=logits.device)
            per_row = torch.stack([t if isinstance(t, torch.Tensor) else torch.full((rows,), float(t), **like) for t in given], 1)
        self.tensors, self.bends = (actions, lengths, per_row), per_row_repetition or repetition != 1.0


def _adjust(x, legal, bias, taken, out):
    x, legal, bias = _unit(x.resolve_neg()), _unit(legal), _unit(bias if bias is None else bias.resolve_neg())
    rows, cols = x.shape
    actions, lengths, per_row = taken.tensors
    stride, history = (0, 0) if actions is None else (actions.stride(0), actions.shape[1])
    _lib.check(_lib.lib().mtaz_adjust_logits(
        x.device.index, rows, cols, TYPES[x.dtype], x.data_ptr(), x.stride(0), out.data_ptr(), out.stride(0),
        _ptr(legal), _row_stride(legal), _ptr(bias), _row_stride(bias), _ptr(actions), stride,
        history, _ptr(lengths), _doubles(*taken.host), _ptr(per_row), _stream(x.device)))
    return out


def adjust_logits(logits, legal=None, bias=None, actions=None, lengths=None, repetition=1.0, frequency=0.0,
                  presence=0.0, out=None):
    """Logits a policy is to answer with.  With c = how often the row has taken action v:

        x <- x / repetition if x > 0 else x * repetition, then x - c frequency - presence   (where c > 0)
        y  = x + bias where v is legal, -inf elsewhere (whatever x holds there)

    legal: packed masks (see the module).  bias: float32 [cols], [1, cols] or [rows, cols].  actions: int32
    [rows, history], of which the first lengths[row] (int32; None: all) count; entries outside [0, cols) (a
    padding of -1, say) do not.  The penalties are numbers or float32 tensors [rows]; repetition must be
    positive.  Where logits or bias require a gradient the result is differentiable; the gradient of a bias that the
    rows share is summed over them in a fixed order.  out (logits itself is allowed): not with gradients."""
    _check_logits(logits)
    rows, cols = logits.shape
    _check_legal(legal, logits)
    if bias is not None:
        _check_rows(bias, 'bias', logits, ((cols,), (1, cols), (rows, cols)), (torch.float32,))
    taken = _Taken(logits, actions, lengths, repetition, frequency, presence)
    if out is None:
        return _call(_lib.nodes().adjust_logits.default, logits, bias, legal, *taken.tensors, *taken.host, taken.bends)
    if torch.is_grad_enabled() and (logits.requires_grad or (bias is not None and bias.requires_grad)):
        raise ValueError('out is not supported where a gradient is required')
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError('out must have the shape, type and device of logits')
    if (cols > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < cols):
        raise ValueError('out must have dense rows that do not overlap')
    if out.is_neg():
        raise ValueError('out must not be a negated view')
    if torch.is_grad_enabled() and out.requires_grad:
        raise ValueError('out must not require a gradient')
    _no_tangent('adjust_logits', logits, bias, taken.tensors[2], out)
    _not_traced('adjust_logits with out')
    _adjust(logits, legal, bias, taken, out)
    torch.autograd.graph.increment_version(out)
    return out


# ---- policy/value loss -------------------------------------------------------------------------------------
def _check_loss(logits, target, value, reward, legal):
    _check_logits(logits)
    rows, cols = logits.shape
    if rows == 0:
        raise ValueError('the mean loss of no rows')
    _check_rows(target, 'target', logits, ((rows, cols),), (torch.float32, logits.dtype))
    if (value is None) != (reward is None):
        raise ValueError('value and reward come together')
    if value is not None:
        shapes = ((rows,), (rows, 1))
        _check_rows(value, 'value', logits, shapes, (torch.float32,))
        _check_rows(reward, 'reward', logits, shapes, (torch.float32,))
    _check_legal(legal, logits)
    if torch.is_grad_enabled() and (target.requires_grad or (reward is not None and reward.requires_grad)):
        raise ValueError('target and reward have no gradient')


def policy_value_loss(logits, target, value=None, reward=None, legal=None):
    """The mean over the rows of (value - reward)^2 - sum over the legal v of target_v log softmax(logits)_v
    (exp/learner.py:86-87, where every action counts as legal), a float32 scalar.

    target: float32 or of the logits' type; it need not sum to 1.  value, reward: float32 [rows] or [rows, 1],
    or neither.  Masked places do not matter, whatever they hold (an output of adjust_logits needs no mask),
    a target of 0 adds nothing, and a row with nothing legal, or with every legal logit at -inf, adds its value term
    alone.  Differentiable in logits and value."""
    _check_loss(logits, target, value, reward, legal)
    return _call(_lib.nodes().policy_loss.default, logits, value, target, reward, legal)[0]


def policy_value_loss_grad(logits, target, value=None, reward=None, legal=None, scale=1.0):
    """policy_value_loss and the gradients of scale * loss, from one pass: (loss, d logits, d value or None),
    for torch.autograd.backward((logits, value), (d logits, d value)); the three are cut off from autograd's graph.
    With 16-bit logits a scale keeps small gradients in range."""
    _check_loss(logits, target, value, reward, legal)
    return _call(_lib.nodes().policy_loss_grad.default, logits, value, target, reward, legal, float(scale))
