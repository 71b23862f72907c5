"""Muon: momentum whose update is orthogonalised, on hand-written HIP kernels (csrc/mtaz_muon.hip).

The reference trains with AdamW alone (exp/learner.py:71-72), and that stays the learner's default.
Muon is the other choice for weights that are matrices: a convolution [out, in, kh, kw] counts as
the matrix [out, in * kh * kw].

    orthogonalize(grad)                   U V^T of grad = U S V^T, roughly, by Newton-Schulz products
    muon_step(params, grads, momenta)     one step on a list of parameters
    Muon(params, lr)                      the same as a torch.optim.Optimizer

Every function enqueues on the current stream of its tensors' device, synchronizes nothing, and may be
captured in a HIP graph (not traced by make_fx: that is refused).  There is no CPU form: tensors elsewhere are refused.
"""
import bisect
import ctypes
import functools
import math

import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import _lib

# X <- a X + (b S + c S S) X, S = X X^T: five steps take singular values in [0.003, 1] to about [0.7, 1.2]
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


@functools.lru_cache(maxsize=64)
def _doubles(*values):
    return (ctypes.c_double * len(values))(*values)


def _coefficients(values):
    values = tuple(float(v) for v in values)
    if len(values) != 3:
        raise ValueError(f'expected three coefficients, got {len(values)}')
    return _doubles(*values)


def _pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def _workspace_size(n, rows, cols, dtype):
    """Bytes of scratch memory; refuses shapes that the kernels do not take."""
    return _lib.check(_lib.lib().mtaz_orthogonalize_workspace(n, rows, cols, TYPES[dtype]))


def _workspace(size, device):
    return torch.empty(size, dtype=torch.uint8, device=device)


def _check_type(t, what):
    if t.device.type != 'cuda':
        raise ValueError(f'{what} must be on a GPU (HIP kernels), not on {t.device}')
    if t.dtype not in TYPES:
        raise ValueError(f'{what} must be float32, float16 or bfloat16, not {t.dtype}')


def _no_tangent(what, *tensors):
    """Refuses tensors that carry a tangent (forward-mode differentiation): the result would have none, which says
    that its derivative is 0."""
    if getattr(forward_ad, '_current_level', 0) < 0:   # no dual level is open
        return
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f'{what} has no forward-mode derivative')


def _not_traced(what):
    """Refuses a call that a tracer (make_fx) would not record: it goes straight to the C entry."""
    if torch._C._len_torch_dispatch_stack() and get_proxy_mode() is not None:
        raise RuntimeError(f'{what} cannot be traced into a graph of torch operators')


def _span(t):
    """The addresses of a contiguous tensor: (first, behind the last)."""
    at = t.data_ptr()
    return at, at + t.numel() * t.element_size()


def _stream(device):
    """The current stream of a device, as the C entries take it."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def orthogonalize(grad, steps=5, coefficients=COEFFICIENTS, eps=1e-7, out=None):
    """Each matrix of grad [..., rows, cols] (float32, float16 or bfloat16) divided by its Frobenius
    norm + eps and taken through `steps` Newton-Schulz steps over its shorter side.  The result has
    grad's type and shape; whatever the type, the products have factors of 22 bits and float32 sums, and
    the result is rounded once.  out: a contiguous tensor for the result (grad itself is allowed).  There is no
    backward pass and no forward-mode derivative.

    Accuracy is relative to the largest singular value: entries below 2^-38 of the norm are taken as 0."""
    _check_type(grad, 'grad')
    if grad.dim() < 2:
        raise ValueError(f'grad must have at least two dimensions, got {tuple(grad.shape)}')
    if torch.is_grad_enabled() and grad.requires_grad:
        raise ValueError('orthogonalize has no backward pass: detach grad')
    _no_tangent('orthogonalize', grad, out)
    _not_traced('orthogonalize')
    if out is None:
        out = torch.empty(grad.shape, dtype=grad.dtype, device=grad.device)
    elif out.shape != grad.shape or out.dtype != grad.dtype or out.device != grad.device or not out.is_contiguous():
        raise ValueError('out must be contiguous and have the shape, type and device of grad')
    elif out.is_neg():
        raise ValueError('out must not be a negated view')
    elif torch.is_grad_enabled() and out.requires_grad:
        raise ValueError('out must not require a gradient')
    rows, cols = grad.shape[-2:]
    n = math.prod(grad.shape[:-2])
    src = grad.detach().resolve_neg().contiguous()   # as it is: torch may hold a negated view of other numbers
    (a, b), (c, d) = _span(src), _span(out)
    if a != c and a < d and c < b:
        raise ValueError('out overlaps grad and is not grad')
    step = rows * cols * src.element_size()
    ptrs, outs = (ctypes.c_void_p * n)(), (ctypes.c_void_p * n)()
    for i in range(n):
        ptrs[i], outs[i] = src.data_ptr() + i * step, out.data_ptr() + i * step
    work = _workspace(_workspace_size(n, rows, cols, grad.dtype), grad.device)
    _lib.check(_lib.lib().mtaz_orthogonalize(
        grad.device.index, n, rows, cols, TYPES[grad.dtype], ptrs, outs, int(steps), _coefficients(coefficients),
        float(eps), work.data_ptr(), work.numel(), _stream(grad.device)))
    torch.autograd.graph.increment_version(out)
    return out


@torch.no_grad()
def muon_step(params, grads, momenta, *, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
              coefficients=COEFFICIENTS, eps=1e-7, scale=None):
    """One Muon step, in place, on parameters of at least two dimensions (rows = the first, cols = the rest):

        m <- momentum m + (1 - momentum) g
        u  = (1 - momentum) g + momentum m  (nesterov)  or  m
        w <- (1 - lr weight_decay) w - lr scale orthogonalize(u)

    scale: a factor, or None for sqrt(max(1, rows / cols)), which keeps the update's effect on a layer's
    outputs alike for tall and wide matrices.  Momenta are float32 tensors of the parameters' shapes.  The
    parameters may differ in shape and type; those alike go through the kernels together."""
    params, grads, momenta = list(params), list(grads), list(momenta)
    if not len(params) == len(grads) == len(momenta):
        raise ValueError(f'{len(params)} parameters, {len(grads)} gradients and {len(momenta)} momenta')
    _no_tangent('muon_step', *params, *grads, *momenta)
    _not_traced('muon_step')
    groups, written, read = {}, [], []
    for w, g, m in zip(params, grads, momenta):
        _check_type(w, 'a parameter')
        if w.dim() < 2 or w.numel() == 0:
            raise ValueError(f'Muon takes parameters of at least two dimensions with elements, got {tuple(w.shape)}')
        if g.shape != w.shape or g.dtype != w.dtype or g.device != w.device or g.layout != torch.strided:
            raise ValueError('a gradient must be dense and have its parameter\'s shape, type and device')
        if m.shape != w.shape or m.dtype != torch.float32 or m.device != w.device:
            raise ValueError('a momentum must be float32 and have its parameter\'s shape and device')
        if not (w.is_contiguous() and m.is_contiguous()):
            raise ValueError('parameters and momenta must be contiguous')
        if w.is_neg() or m.is_neg():
            raise ValueError('parameters and momenta must not be negated views')
        g = g.resolve_neg().contiguous()
        written += _span(w), _span(m)
        if _span(g) != _span(w):   # a gradient in its own parameter's place has been read when that is written
            read.append(_span(g))
        groups.setdefault((w.device, w.dtype, w.shape[0], w.numel() // w.shape[0]), []).append((w, g, m))
    written.sort()
    for (_, end), (start, _) in zip(written, written[1:]):
        if start < end:
            raise ValueError('the same parameter or momentum twice in one step, or two that overlap')
    for start, end in read:   # the written spans do not overlap: the last one that starts before `end` decides
        at = bisect.bisect_left(written, (end,))
        if at and written[at - 1][1] > start:
            raise ValueError('a gradient overlaps a parameter or a momentum')
    co = _coefficients(coefficients)
    # all shapes are looked at before the first group's step
    sizes = [_workspace_size(len(group), rows, cols, dtype) for (_, dtype, rows, cols), group in groups.items()]
    for ((device, dtype, rows, cols), group), size in zip(groups.items(), sizes):
        ws, gs, ms = zip(*group)
        work = _workspace(size, device)
        factor = math.sqrt(max(1.0, rows / cols)) if scale is None else float(scale)
        _lib.check(_lib.lib().mtaz_muon_step(
            device.index, len(ws), rows, cols, TYPES[dtype], _pointers(ws), _pointers(gs), _pointers(ms), float(lr),
            float(momentum), int(bool(nesterov)), float(weight_decay), factor, int(steps), co, float(eps),
            work.data_ptr(), work.numel(), _stream(device)))
        torch.autograd.graph.increment_version(ws + ms)   # a graph that saved them must notice


class Muon(torch.optim.Optimizer):
    """muon_step as an optimizer.  Give it the weights that are matrices (hidden layers); embeddings,
    heads, biases and norms train better with AdamW (learner.muon_split divides a network).  The
    momenta are float32 whatever the parameters' type, in the state as 'momentum_buffer'; the first step makes
    them, so it is not one to capture in a graph.  A captured step keeps the lr and the other numbers of its capture."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
                 coefficients=COEFFICIENTS, eps=1e-7, scale=None):
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f'momentum must be in [0, 1), got {momentum}')
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      steps=steps, coefficients=tuple(coefficients), eps=eps, scale=scale))
        for group in self.param_groups:
            for p in group['params']:
                if p.dim() < 2:
                    raise ValueError(f'Muon takes parameters of at least two dimensions, got {tuple(p.shape)}')

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group['params'] if p.grad is not None]
            for p in params:
                if not self.state[p]:
                    if torch.cuda.is_current_stream_capturing():   # a replay would set the momentum to 0 again
                        raise RuntimeError('the first step of a parameter cannot be captured: run one before the capture')
                    self.state[p]['momentum_buffer'] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            muon_step(params, [p.grad for p in params], [self.state[p]['momentum_buffer'] for p in params],
                      **{k: group[k] for k in ('lr', 'momentum', 'nesterov', 'weight_decay', 'steps', 'coefficients',
                                               'eps', 'scale')})
        return loss

    def load_state_dict(self, state_dict):
        """torch's, with the momenta put back in float32 (torch casts a state to its parameter's type)."""
        super().load_state_dict(state_dict)
        ours = [p for g in self.param_groups for p in g['params']]
        theirs = [i for g in state_dict['param_groups'] for i in g['params']]
        for p, i in zip(ours, theirs):
            saved = state_dict['state'].get(i, {}).get('momentum_buffer')
            if saved is not None:
                self.state[p]['momentum_buffer'] = saved.detach().to(p.device, torch.float32, copy=True).contiguous()
