"""The network itself, next to its bounds: fc layers forward and backward, the
classification loss with its gradient, and the optimiser's step, on the library's
kernels (no reference counterpart).

Tensors are fp32 or bf16 on the GPU; every function runs on the current stream,
allocates its outputs and workspace from torch and waits for nothing.  CPU tensors
raise RuntimeError, other types NotImplementedError, sizes that do not fit
ValueError.

Gradients are first derivatives in reverse mode: a second derivative (through what
create_graph=True returned) and forward mode (a dual tensor) raise NotImplementedError.
What is written in place counts as written: a graph that saved it raises when it is used.
"""
import math
import operator
from array import array

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from ._lib import call, load, stream

ACTS = {None: 0, 'none': 0, 'relu': 1, 'gelu': 2, 'silu': 3}
REDUCTIONS = {'none': 0, 'sum': 1, 'mean': 2}
BLOCK = 256     # values of an optimiser state that share a scale
E4M3_MAX = 448.0
_DZ_ROUNDED = 16    # or'ed to a backward's activation
_TYPES = {torch.float32: 0, torch.bfloat16: 1}


def _type(t, what):
    """The library's number for a GPU tensor's type."""
    if not t.is_cuda:
        raise RuntimeError(f'vibecheck_amd: {what} is not on the GPU '
                           '(the HIP library is the only compute path)')
    k = _TYPES.get(t.dtype)
    if k is None:
        raise NotImplementedError(f'vibecheck_amd: {what} is {t.dtype}; fp32 and bf16 are taken')
    if t.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f'vibecheck_amd: {what} is on {t.device}, not on the current device')
    return k


def _no_tangents(*tensors):
    """Forward-mode derivatives would be lost without a word."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError('vibecheck_amd: the kernels have no forward-mode derivative')


class _First(torch.autograd.Function):
    """Passes on what follows n tensors that it depends on; a derivative of it raises."""
    @staticmethod
    def forward(ctx, n, *tensors):
        return tensors[n:]

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError('vibecheck_amd: the kernels have no second derivative')


def _first(grads, *on):
    """What a backward gives: under create_graph=True no constant, but dependent on ``on``."""
    return _First.apply(len(on), *on, *grads) if torch.is_grad_enabled() else grads


def _like(t, ref, shape, what):
    if t.dtype != ref.dtype or t.get_device() != ref.get_device():
        raise ValueError(f'vibecheck_amd: {what} is {t.dtype} on {t.device}, '
                         f'expected {ref.dtype} on {ref.device}')
    if t.shape != shape:
        raise ValueError(f'vibecheck_amd: {what} has shape {tuple(t.shape)}, '
                         f'expected {tuple(shape)}')


def _rows(t):
    """t as rows of its last axis, values of a row side by side: (tensor to keep, row stride)."""
    n = t.shape[-1]
    if t.is_contiguous():
        return t, n
    if t.dim() != 2:
        t = t.reshape(-1, n)
    if t.shape[0] <= 1 or n == 0:
        return t.contiguous(), n
    if t.stride(1) != 1 and n > 1 or t.stride(0) < n:
        t = t.contiguous()
    return t, t.stride(0)


def _lead(t, n):
    """Rows of t's last axis, and t's shape with n in place of it."""
    if t.dim() == 2:
        M = t.shape[0]
        return M, (M, n)
    lead = tuple(t.shape[:-1])
    return math.prod(lead), lead + (n,)


def _ptr(t):
    return None if t is None else t.data_ptr()


_sizes = {}  # (function, its arguments): the bytes it gave


def _work(like, name, *args):
    """(tensor to keep or None, its pointer, its bytes) of a call's workspace."""
    n = _sizes.get((name, args))
    if n is None:
        n = getattr(load(), name)(*args)
        if n < 0:
            raise ValueError('vibecheck_amd: sizes out of range')
        if len(_sizes) > 4096:
            _sizes.clear()
        _sizes[name, args] = n
    if n == 0:
        return None, None, 0
    t = torch.empty(n, dtype=torch.uint8, device=like.device)
    return t, t.data_ptr(), n


# ------------------------------------------------------------------- fc layer

def _act(act):
    if act not in ACTS:
        raise ValueError(f'vibecheck_amd: activation {act!r}; one of {list(ACTS)} is taken')
    return ACTS[act]


def _linear(x, W, bias, act, residual, save):
    k = _type(x, 'x')
    if x.dim() < 1 or W.dim() != 2:
        raise ValueError('vibecheck_amd: x has at least one axis, W two')
    N, K = W.shape
    _like(W, x, (N, x.shape[-1]), 'W')
    M, shape = _lead(x, N)
    if bias is not None:
        _like(bias, x, (N,), 'bias')
        bias = bias.contiguous()
    if residual is not None:
        _like(residual, x, shape, 'residual')
    x, ldx = _rows(x)
    W = W.contiguous()
    y = x.new_empty(shape)
    # the sign of relu's output is its input's; another activation's input is kept
    z = torch.empty_like(y) if save and act and (act != 1 or residual is not None) else None
    if residual is not None:
        residual, ldr = _rows(residual)
    else:
        ldr = 0
    work, at, nbytes = _work(x, 'vc_linear_workspace', k, M, K, N)
    call('vc_linear', k, x.data_ptr(), M, K, ldx, W.data_ptr(), N, _ptr(bias), act,
         _ptr(residual), ldr, y.data_ptr(), _ptr(z), at, nbytes, stream())
    return y, (y if save and act and z is None else z)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, W, bias, act, residual, round_dz):
        y, z = _linear(x, W, bias, act, residual, True)
        ctx.save_for_backward(x, W, z)
        ctx.act, ctx.round_dz, ctx.bias = act, round_dz, bias
        return y

    @staticmethod
    def backward(ctx, dy):
        x, W, z = ctx.saved_tensors
        needs = ctx.needs_input_grad
        need = [n for n, on in zip(('x', 'W', 'bias'), needs) if on]
        dx = dW = db = None
        if need:
            dx, dW, db = _first(linear_backward(dy, x, W, z, ctx.act, need, ctx.round_dz),
                                dy, x, W, ctx.bias)
        return dx, dW, db, None, dy if needs[4] else None, None


def linear(x, W, bias=None, act=None, residual=None, save=False, round_dz=False):
    """act(x W^T + bias) + residual for x (..., K), W (N, K), bias (N), residual (..., N), all of
    one type.  ``act``: None, 'relu', 'gelu' (the erf form) or 'silu'.

    Differentiable through autograd for inputs that require it; ``round_dz`` is what
    linear_backward is then given.  With ``save`` it returns (y, z) instead, outside of any
    graph, z what the caller gives to linear_backward (None without an activation; for relu
    without a residual it is y itself)."""
    a = _act(act)
    _no_tangents(x, W, bias, residual)
    if not save and torch.is_grad_enabled() and (
            x.requires_grad or W.requires_grad or bias is not None and bias.requires_grad or
            residual is not None and residual.requires_grad):
        return _Linear.apply(x, W, bias, a, residual, round_dz)
    y, z = _linear(x, W, bias, a, residual, save)
    return (y, z) if save else y


_ALL = ('x', 'W', 'bias')


def linear_backward(dy, x, W, z=None, act=None, need=_ALL, round_dz=False):
    """(dx, dW, db) of y = act(x W^T + bias) from dy (..., N): dz = dy act'(z), dx = dz W,
    dW = dz^T x, db the sum of dz over rows; None for what ``need`` does not name.  ``z`` is
    what linear(save=True) returned.  The residual's gradient is dy.

    The bf16 products of a GELU's or SiLU's dz take it in two parts, at twice their work, so that
    dx and dW are off by their own rounding alone (1.7e-3 of their norm).  ``round_dz`` rounds
    it to bf16 first (2.3e-3); it changes nothing for the other activations or in fp32."""
    a = act if isinstance(act, int) else _act(act)
    _no_tangents(dy, x, W, z)
    k = _type(dy, 'dy')
    if W.dim() != 2 or dy.dim() < 1:
        raise ValueError('vibecheck_amd: dy has at least one axis, W two')
    if need is not _ALL and not set(need) <= set(_ALL):
        raise ValueError(f"vibecheck_amd: need names {need!r}; 'x', 'W' and 'bias' are taken")
    N, K = W.shape
    _like(W, dy, (dy.shape[-1], K), 'W')
    M, of_x = _lead(dy, K)
    _like(x, dy, of_x, 'x')
    if a:
        if z is None:
            raise ValueError('vibecheck_amd: an activation needs z')
        _like(z, dy, dy.shape, 'z')
        z, ldz = _rows(z)
    else:
        z, ldz = None, 0
    dx = dy.new_empty(of_x) if 'x' in need else None
    dW = dy.new_empty((N, K)) if 'W' in need else None
    # no row adds to it, no launch writes it
    db = (dy.new_empty if M else dy.new_zeros)(N) if 'bias' in need else None
    dy, ldy = _rows(dy)
    x, ldx = _rows(x)
    W = W.contiguous()
    which = (dx is not None) + 2 * (dW is not None) + 4 * (db is not None)
    if round_dz:
        a += _DZ_ROUNDED
    work, at, nbytes = _work(dy, 'vc_linear_backward_workspace', k, M, K, N, a, which)
    call('vc_linear_backward', k, dy.data_ptr(), ldy, x.data_ptr(), ldx, W.data_ptr(), _ptr(z), ldz,
         a, M, K, N, _ptr(dx), _ptr(dW), _ptr(db), at, nbytes, stream())
    return dx, dW, db


# ----------------------------------------------------------------------- loss

class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tie, target, reduction, ignore_index, smoothing):
        loss, d = _cross_entropy(logits, target, reduction, ignore_index, smoothing, True, None)
        ctx.save_for_backward(d)
        ctx.tie = tie
        ctx.mark_non_differentiable(d)
        return loss, d

    @staticmethod
    def backward(ctx, g, _):
        d, = _first(ctx.saved_tensors, ctx.tie)
        return (d * g.unsqueeze(-1) if g.dim() else d * g).to(d.dtype), None, None, None, None, None


class _LossAlone(torch.autograd.Function):
    """The gradient computed when it is asked for."""
    @staticmethod
    def forward(ctx, logits, target, *how):
        ctx.save_for_backward(logits, target)
        ctx.how = how
        return _cross_entropy(logits, target, *how, False, None)[0]

    @staticmethod
    def backward(ctx, g):
        logits, target = ctx.saved_tensors
        d, = _first(_cross_entropy(logits, target, *ctx.how, True, None)[1:], logits)
        return (d * g.unsqueeze(-1) if g.dim() else d * g).to(d.dtype), None, None, None, None


def _cross_entropy(logits, target, reduction, ignore_index, smoothing, grad, out):
    k = _type(logits, 'logits')
    if reduction not in REDUCTIONS:
        raise ValueError(f'vibecheck_amd: reduction {reduction!r}; one of {list(REDUCTIONS)} is taken')
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError('vibecheck_amd: logits have at least one class')
    if not 0 <= smoothing <= 1:
        raise ValueError(f'vibecheck_amd: smoothing {smoothing} is not in [0, 1]')
    lead, V = logits.shape[:-1], logits.shape[-1]
    if target.dtype != torch.int64 or target.get_device() != logits.get_device() or target.shape != lead:
        raise ValueError(f'vibecheck_amd: target is {target.dtype} {tuple(target.shape)} on '
                         f'{target.device}, expected int64 {tuple(lead)} on {logits.device}')
    R, kind = lead.numel(), REDUCTIONS[reduction]
    loss = logits.new_empty(lead if kind == 0 else (), dtype=torch.float32)
    if out is not None:
        _like(out, logits, logits.shape, 'out')
        if not out.is_contiguous():
            raise ValueError('vibecheck_amd: out must be contiguous')
        d = out
    else:
        d = logits.new_empty(logits.shape) if grad else None
    z, ld = _rows(logits)
    if out is not None and R > 0:
        # row for row it may be the logits; shifted, a row would be read after it was written
        at, to, e = z.data_ptr(), out.data_ptr(), out.element_size()
        if (at != to or ld != V and R > 1) and to < at + ((R - 1) * ld + V) * e and at < to + R * V * e:
            raise ValueError('vibecheck_amd: out overlaps the logits without being them')
    target = target.contiguous()
    work, at, nbytes = _work(logits, 'vc_cross_entropy_workspace', R, kind)
    call('vc_cross_entropy', k, z.data_ptr(), R, V, ld, target.data_ptr(), ignore_index, smoothing,
         kind, loss.data_ptr(), _ptr(d), V, at, nbytes, stream())
    if out is not None:
        increment_version(out)
    return loss, d


def cross_entropy(logits, target, reduction='mean', ignore_index=-100, smoothing=0.0, grad=True,
                  out=None):
    """(loss, dlogits) of softmax cross-entropy: logits (..., V), target int64 (...), loss fp32,
    dlogits of the logits' type (None without ``grad``; written to ``out``, which may be the
    logits, where that is given).

    loss = lse - (1 - smoothing) z_t - smoothing mean(z) per row ('none'), summed, or averaged
    over the rows whose target is not ``ignore_index``; dlogits is its gradient (per row for
    'none').  A target that is no class gives NaN, a row without a logit above -inf an infinite
    loss and no gradient.  The loss is differentiable where the logits require it; with ``out``
    it is not: the gradient is there to be passed on (logits.backward(out))."""
    _no_tangents(logits)
    if torch.is_grad_enabled() and logits.requires_grad and out is None:
        if not grad:
            return _LossAlone.apply(logits, target, reduction, ignore_index, smoothing), None
        # no value of the logits, but their place in the graph: the node need not keep them
        tie = logits[..., :0].clone()
        return _Loss.apply(logits, tie, target, reduction, ignore_index, smoothing)
    return _cross_entropy(logits, target, reduction, ignore_index, smoothing, grad, out)


# ------------------------------------------------------------------ optimiser

def _blocks(params):
    return sum((p.numel() + BLOCK - 1) // BLOCK for p in params)


def adamw_state(params, bits=32):
    """A new state for adamw_step over ``params``: {'bits', 'm', 'v'} of fp32 values, each tensor
    padded to blocks of 256, or with ``bits`` 8 the bytes of e4m3 values ('m', and in 'v' the
    square roots) and one scale per block ('m_scale', 'v_scale')."""
    if bits not in (8, 32):
        raise ValueError(f'vibecheck_amd: states of {bits} bits; 8 and 32 are taken')
    params = list(params)
    n = _blocks(params)
    dev = params[0].device if params else 'cuda'
    if bits == 32:
        return {'bits': 32, 'm': torch.zeros(n * BLOCK, device=dev),
                'v': torch.zeros(n * BLOCK, device=dev)}
    return {'bits': 8, 'm': torch.zeros(n * BLOCK, dtype=torch.uint8, device=dev),
            'v': torch.zeros(n * BLOCK, dtype=torch.uint8, device=dev),
            'm_scale': torch.zeros(n, device=dev), 'v_scale': torch.zeros(n, device=dev)}


def adamw_moments(params, state):
    """[(m, v), ...] of each parameter in fp32, from a state of either kind."""
    m, v = state['m'], state['v']
    if state['bits'] == 8:
        m, v = ((c.view(torch.float8_e4m3fn).float().view(-1, BLOCK) * s.unsqueeze(1)).view(-1)
                for c, s in ((m, state['m_scale']), (v, state['v_scale'])))
        v = v * v
    out, at = [], 0
    for p in params:
        out.append(tuple(t[at:at + p.numel()].view(p.shape) for t in (m, v)))
        at += (p.numel() + BLOCK - 1) // BLOCK * BLOCK
    return out


_numel, _data_ptr = torch.Tensor.numel, torch.Tensor.data_ptr
_device_of, _contiguous = torch.Tensor.get_device, torch.Tensor.is_contiguous
_dtype_of = operator.attrgetter('dtype')


def _one_type(tensors, sizes, what):
    """Type number and pointers of a list of contiguous GPU tensors of one type."""
    k, n = _type(tensors[0], what), len(tensors)
    if list(map(_dtype_of, tensors)).count(tensors[0].dtype) != n or \
            list(map(_device_of, tensors)).count(tensors[0].get_device()) != n or \
            list(map(_numel, tensors)) != sizes or not all(map(_contiguous, tensors)):
        raise ValueError(f'vibecheck_amd: {what} are contiguous, of one type, on one device and '
                         f'of their parameters\' sizes {sizes}; got '
                         f'{[(t.dtype, str(t.device), tuple(t.shape)) for t in tensors]}')
    return k, array('Q', map(_data_ptr, tensors))


def adamw_step(params, grads, state, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=0.01, copies=None, scale=None):
    """One AdamW step in place, all tensors by one launch per 88: params (fp32 or bf16), grads
    (fp32 or bf16), ``state`` from adamw_state, ``step`` counting from 1, with
    torch.optim.AdamW's formula.  ``copies``: bf16 tensors that receive the new parameters.  ``scale``: one fp32
    value on the GPU that multiplies the gradients (a clip, a loss scale); where it is not finite
    the step changes nothing.

    States of 8 bits are rounded up or down by a hash of the value's place and the step, so that
    a step that moves a value by less than its grid does move it on average; the same inputs
    give the same results."""
    params, grads = list(params), list(grads)
    if not params:
        return
    sizes = list(map(_numel, params))
    if len(grads) != len(params) or (copies is not None and len(copies) != len(params)):
        raise ValueError('vibecheck_amd: one gradient (and copy) for each parameter')
    kp, pp = _one_type(params, sizes, 'params')
    kg, pg = _one_type(grads, sizes, 'grads')
    dev = params[0].get_device()  # the current one, as the gradients' and copies' is
    n, cnt = sum([(k + BLOCK - 1) // BLOCK for k in sizes]), len(sizes)
    bits = state['bits']
    keys = ('m', 'v') if bits == 32 else ('m', 'v', 'm_scale', 'v_scale')
    for key in keys:
        t = state[key]
        want = torch.float32 if bits == 32 or key[1:] else torch.uint8
        if t.dtype != want or t.numel() != (n if key[1:] else n * BLOCK) or \
                t.get_device() != dev or not t.is_contiguous():
            raise ValueError(f'vibecheck_amd: state {key!r} does not fit these parameters')
    if copies is not None:
        kc, pc = _one_type(copies, sizes, 'copies')
        if kc != 1:
            raise ValueError('vibecheck_amd: copies are bf16 tensors beside their parameters')
    if scale is not None and (scale.dtype != torch.float32 or scale.numel() != 1 or
                              scale.get_device() != dev):
        raise ValueError('vibecheck_amd: scale is one fp32 value on the parameters\' device')
    pn = array('q', sizes)
    call('vc_adamw_step', pp.buffer_info()[0], pg.buffer_info()[0],
         None if copies is None else pc.buffer_info()[0], pn.buffer_info()[0], cnt, kp, kg, bits,
         state['m'].data_ptr(), state['v'].data_ptr(), _ptr(state.get('m_scale')),
         _ptr(state.get('v_scale')), lr, betas[0], betas[1], eps, weight_decay, step, _ptr(scale),
         stream())
    increment_version(params + [state[k] for k in keys] + list(copies or ()))
