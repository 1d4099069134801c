"""Operators on GPU tensors for sequence layers and their training, as hand-written HIP kernels (csrc/k_decay.hip,
csrc/k_distill.hip behind include/pxg.h).

  decay_attention        a recurrent layer whose time axis is not serial: linear attention with one decay per head, whole
                         (padded, ragged) batches, differentiable; what an LSTM layer is to ``training`` otherwise
  decay_attention_step   the same recurrence for one more step of many streams, the states updated in place
  top_logits             a teacher network's largest logits per row, with the log-sum-exp of all others
  distillation_loss      the loss of a student's logits against them, differentiable: with it the networks this package ships
                         teach others (``training.Trainer`` takes it as its ``loss_fn``)

Tensors live on one GPU; calls run on the current stream of that GPU and return without waiting.  They only launch kernels, so
they may be captured into a graph.  The library missing or a tensor on another device raises: there is no fallback.
"""
import ctypes as C

import torch

from . import native as _native

__all__ = ['TopLogits', 'decay_attention', 'decay_attention_backward', 'decay_attention_step', 'distillation_loss',
           'distillation_loss_and_gradient', 'top_logits', 'MAX_WIDTH', 'MAX_K']

MAX_WIDTH = _native.PXG_DECAY_MAX_WIDTH
MAX_K = _native.PXG_TOP_MAX_K

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}          # enum pxg_dtype
_EAGER_STREAM = 'pxg_eager_stream'


# ---- checks and calls ---------------------------------------------------------------------------------------------
def _on_gpu(name, t, device=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError('{} must be a tensor, not {}'.format(name, type(t).__name__))
    if not t.is_cuda:
        raise ValueError('{} is on {}: these operators run on a GPU only'.format(name, t.device))
    if device is not None and t.device != device:
        raise ValueError('{} is on {}, the other tensors are on {}'.format(name, t.device, device))


def _floats(name, t):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError('{} is {}: float32, bfloat16 or float16 is needed'.format(name, t.dtype))
    return code


def _f32(name, t, shape, device):
    _on_gpu(name, t, device)
    if t.dtype != torch.float32:
        raise TypeError('{} is {}: float32 is needed'.format(name, t.dtype))
    if tuple(t.shape) != shape:
        raise ValueError('{} has shape {}, {} is needed'.format(name, tuple(t.shape), shape))


def _call(fn, struct, device):
    """Launch on the current stream of `device` (and with it as the current device: kernels go where their data is)."""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _call(fn, struct, device)
    rc = fn(C.byref(struct), torch._C._cuda_getCurrentRawStream(device.index))
    if rc:
        _fail(fn.__name__, rc)


def _fail(what, rc):
    raise _native.PxgError('{} failed ({})'.format(what, rc))


def _lib():
    return _native._lib or _native.load_library()


def _differentiable(function, leaves, *args):
    """function.apply(*args).  The gradient of a leaf is accumulated on the stream where its oldest living graph was built.  Captured
    on another stream, the backward pass would have to wait for that stream from inside the capture, which ends the process:
    refused here instead.  (The mark lives and dies with the graphs that hold it.)"""
    leaves = [t for t in leaves if t is not None and t.requires_grad and t.grad_fn is None]
    stream = torch._C._cuda_getCurrentRawStream(args[1].device.index)
    capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        for t in leaves:
            if torch.autograd.graph.get_gradient_edge(t).node.metadata.get(_EAGER_STREAM, stream) != stream:
                raise RuntimeError('capturing a differentiable call while a graph of the same leaf, built on another stream outside '
                                   'the capture, is alive: free that graph first, or capture decay_attention_backward / '
                                   'distillation_loss_and_gradient, which need no autograd graph')
    result = function.apply(*args)
    if not capturing:
        for t in leaves:
            torch.autograd.graph.get_gradient_edge(t).node.metadata.setdefault(_EAGER_STREAM, stream)
    return result


# ---- decay attention ----------------------------------------------------------------------------------------------
def _sequence(t):
    s = t.stride()
    return _native.PxgSequence(t.data_ptr(), s[0], s[1], s[2])


def _rows(t):
    """The kernels take any strides but that of the width."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check_decay(q, k, v, log_decay, lengths, initial_state, steps_axis=True):
    _on_gpu('q', q)
    code, device = _floats('q', q), q.device
    axes = '[batch, steps, heads, width]' if steps_axis else '[batch, heads, width]'
    for name, t in (('k', k), ('v', v)):
        _on_gpu(name, t, device)
        if t.dtype != q.dtype:
            raise TypeError('{} is {}, q is {}'.format(name, t.dtype, q.dtype))
    if q.dim() != (4 if steps_axis else 3) or k.shape != q.shape or v.dim() != q.dim() or v.shape[:-1] != q.shape[:-1]:
        raise ValueError('q, k and v must be {} with equal widths of q and k: got {}, {}, {}'.format(
            axes, tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    batch, heads, dk, dv = q.shape[0], q.shape[-2], q.shape[-1], v.shape[-1]
    if not (1 <= dk <= MAX_WIDTH and 1 <= dv <= MAX_WIDTH and heads >= 1):
        raise ValueError('{} heads of widths {} and {}: at least one head, widths of 1 to {}'.format(heads, dk, dv, MAX_WIDTH))
    _f32('log_decay', log_decay, (heads,), device)
    if lengths is not None:
        _on_gpu('lengths', lengths, device)
        if lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError('lengths is {}: int32 or int64 is needed'.format(lengths.dtype))
        if tuple(lengths.shape) != (batch,):
            raise ValueError('lengths has shape {}, {} is needed'.format(tuple(lengths.shape), (batch,)))
    if initial_state is not None:
        _f32('initial_state', initial_state, (batch, heads, dk, dv), device)
    return code


def _decay_struct(code, q, k, v, log_decay, lengths, initial_state):
    """(the call, what has to stay alive until it was made)"""
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    s = _native.PxgDecay()
    s.struct_bytes = C.sizeof(s)
    s.dtype, s.batch, s.steps, s.heads = code, q.shape[0], q.shape[1], q.shape[2]
    s.dk, s.dv = q.shape[3], v.shape[3]
    s.q, s.k, s.v = _sequence(q), _sequence(k), _sequence(v)
    s.log_decay = log_decay.data_ptr()
    if lengths is not None:
        lengths = lengths.contiguous()
        s.lengths, s.lengths_are_64 = lengths.data_ptr(), int(lengths.dtype == torch.int64)
    if initial_state is not None:
        initial_state = initial_state.contiguous()
        s.initial_state = initial_state.data_ptr()
    return s, (q, k, v, log_decay, lengths, initial_state)


def _workspace(s, backward, device):
    n = _lib().pxg_decay_workspace_bytes(C.byref(s), backward)
    if n < 0:
        _fail('pxg_decay_workspace_bytes', n)
    t = torch.empty(n, dtype=torch.uint8, device=device) if n else None
    if n:
        s.workspace, s.workspace_bytes = t.data_ptr(), n
    return t


def _decay_forward(code, q, k, v, log_decay, lengths, initial_state, want_state):
    s, keep = _decay_struct(code, q, k, v, log_decay, lengths, initial_state)
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    s.out = out.data_ptr()
    state = None
    if want_state:
        state = torch.empty((s.batch, s.heads, s.dk, s.dv), dtype=torch.float32, device=v.device)
        s.final_state = state.data_ptr()
    work = _workspace(s, 0, v.device)
    _call(_lib().pxg_decay_forward, s, v.device)
    del keep, work
    return out, state


def _decay_backward(code, q, k, v, log_decay, lengths, initial_state, grad_out, grad_state, want_decay, want_state):
    s, keep = _decay_struct(code, q, k, v, log_decay, lengths, initial_state)
    grad_out = _rows(grad_out)
    s.grad_out = _sequence(grad_out)
    if grad_state is not None:
        grad_state = grad_state.contiguous()
        s.grad_final_state = grad_state.data_ptr()
    new = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v)]
    s.grad_q, s.grad_k, s.grad_v = (t.data_ptr() for t in new)
    grad_decay = grad_initial = None
    if want_decay:
        grad_decay = torch.empty_like(log_decay, memory_format=torch.contiguous_format)
        s.grad_log_decay = grad_decay.data_ptr()
    if want_state:
        grad_initial = torch.empty((s.batch, s.heads, s.dk, s.dv), dtype=torch.float32, device=q.device)
        s.grad_initial_state = grad_initial.data_ptr()
    work = _workspace(s, 1, q.device)
    _call(_lib().pxg_decay_backward, s, q.device)
    del keep, work
    return new[0], new[1], new[2], grad_decay, grad_initial


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, code, q, k, v, log_decay, lengths, initial_state, want_state):
        out, state = _decay_forward(code, q, k, v, log_decay, lengths, initial_state, want_state)
        ctx.save_for_backward(q, k, v, log_decay, lengths, initial_state)
        ctx.code = code
        ctx.set_materialize_grads(False)
        return out, state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out, grad_state):
        q, k, v, log_decay, lengths, initial_state = ctx.saved_tensors
        need = ctx.needs_input_grad
        if grad_out is None and grad_state is None:
            return (None,) * 8
        if grad_out is None:
            grad_out = torch.zeros((), dtype=v.dtype, device=v.device).expand(v.shape).contiguous()
        gq, gk, gv, gd, gs = _decay_backward(ctx.code, q, k, v, log_decay, lengths, initial_state, grad_out, grad_state,
                                             need[4], need[6])
        return (None, gq if need[1] else None, gk if need[2] else None, gv if need[3] else None, gd, None, gs, None)


def decay_attention(q, k, v, log_decay, lengths=None, initial_state=None, return_state=False):
    """Linear attention with one decay per head over whole sequences.

        S_t = exp(log_decay[h]) S_(t-1) + k_t v_t^T,    o_t = q_t S_t

    q, k [batch, steps, heads, dk] and v [batch, steps, heads, dv], float32, bfloat16 or float16, dk and dv of 1 to 128, any
    strides (k and v that heads share are ``expand``-ed views); log_decay [heads] float32 (-inf: no memory).  lengths [batch]
    (int32 or int64): the steps of each sequence; what lies behind them is not read, and its rows of the result are 0.
    initial_state [batch, heads, dk, dv] float32: S before the first step, 0 if None.

    Returns o [batch, steps, heads, dv] in v's type, or (o, S behind each sequence's last step, float32).  Differentiable in q,
    k, v, log_decay and initial_state.  Sums and states are held in float32 whatever the tensors' type."""
    code = _check_decay(q, k, v, log_decay, lengths, initial_state)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, log_decay, initial_state)):
        out, state = _differentiable(_DecayAttention, (q, k, v, log_decay, initial_state),
                                     code, q, k, v, log_decay, lengths, initial_state, return_state)
    else:
        out, state = _decay_forward(code, q, k, v, log_decay, lengths, initial_state, return_state)
    return (out, state) if return_state else out


def decay_attention_backward(grad_out, q, k, v, log_decay, lengths=None, initial_state=None, grad_state=None):
    """The gradients of decay_attention without an autograd graph (for a captured training step): grad_out like its result and
    grad_state like its state (or None) -> gradients of q, k, v, log_decay and initial_state (None without one)."""
    code = _check_decay(q, k, v, log_decay, lengths, initial_state)
    _on_gpu('grad_out', grad_out, q.device)
    if grad_out.dtype != v.dtype or grad_out.shape != v.shape:
        raise ValueError('grad_out is {} {}, v is {} {}'.format(grad_out.dtype, tuple(grad_out.shape), v.dtype, tuple(v.shape)))
    if grad_state is not None:
        _f32('grad_state', grad_state, (q.shape[0], q.shape[2], q.shape[3], v.shape[3]), q.device)
    with torch.no_grad():
        return _decay_backward(code, q, k, v, log_decay, lengths, initial_state, grad_out, grad_state, True,
                               initial_state is not None)


def decay_attention_step(q, k, v, log_decay, state, active=None):
    """One more step of many streams: q, k [batch, heads, dk], v [batch, heads, dv], state [batch, heads, dk, dv] float32,
    contiguous, updated IN PLACE.  Returns o [batch, heads, dv] in v's type.  active [batch] bool: the state of a stream that is
    not active stays as it is, and its row of the result is 0.  For inference: no gradients."""
    code = _check_decay(q, k, v, log_decay, None, state, steps_axis=False)
    device = q.device
    if not state.is_contiguous():
        raise ValueError('state must be contiguous: it is updated in place')
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, log_decay, state)):
        raise RuntimeError('decay_attention_step has no gradients: call it under torch.no_grad(), or use decay_attention')
    s, keep = _decay_struct(code, q.unsqueeze(1), k.unsqueeze(1), v.unsqueeze(1), log_decay, None, None)
    if active is not None:
        _on_gpu('active', active, device)
        if active.dtype != torch.bool or tuple(active.shape) != (q.shape[0],):
            raise ValueError('active must be bool [{}]: got {} {}'.format(q.shape[0], active.dtype, tuple(active.shape)))
        active = active.contiguous()
        s.lengths = active.data_ptr()
    out = torch.empty(v.shape, dtype=v.dtype, device=device)
    s.out, s.final_state = out.data_ptr(), state.data_ptr()
    _call(_lib().pxg_decay_step, s, device)
    torch.autograd.graph.increment_version(state)
    return out


# ---- learning from a teacher ----------------------------------------------------------------------------------------
class TopLogits:
    """A teacher's answers for many rows: values [rows, k] (descending), indices [rows, k] (their classes; -1: an empty place),
    rest [rows] float32 = log sum over all other classes of exp(logit / temperature), or None: the listed classes are all
    there is.  Rows are picked by indexing, so it serves as the targets of ``training.Trainer.fit``."""

    __slots__ = ('values', 'indices', 'rest', 'temperature')

    def __init__(self, values, indices, rest=None, temperature=1.0):
        self.values, self.indices, self.rest, self.temperature = values, indices, rest, float(temperature)

    def __len__(self):
        return len(self.values)

    def __getitem__(self, rows):
        if isinstance(rows, int):
            rows = slice(rows, rows + 1 or None)
        return TopLogits(self.values[rows], self.indices[rows], None if self.rest is None else self.rest[rows], self.temperature)

    def to(self, *args, **kwargs):
        device = torch.empty(0).to(*args, **kwargs).device          # moves, never casts
        return TopLogits(self.values.to(device), self.indices.to(device), None if self.rest is None else self.rest.to(device),
                         self.temperature)

    @staticmethod
    def cat(parts):
        parts = list(parts)
        rest = None if any(p.rest is None for p in parts) else torch.cat([p.rest for p in parts])
        if len({p.temperature for p in parts}) != 1:
            raise ValueError('answers of different temperatures')
        return TopLogits(torch.cat([p.values for p in parts]), torch.cat([p.indices for p in parts]), rest, parts[0].temperature)


def _temperature(temperature):
    temperature = float(temperature)
    if not 0.0 < temperature <= 3.0e38:
        raise ValueError('temperature is {}: a positive number is needed'.format(temperature))
    return temperature


def top_logits(logits, k, temperature=1.0):
    """The k largest logits of each row (logits [rows, classes], k of 1 to 128) as TopLogits: descending, ties to the lowest
    class, NaN before all numbers; `rest` sums up the other classes at this temperature.  No gradients."""
    _on_gpu('logits', logits)
    code, temperature = _floats('logits', logits), _temperature(temperature)
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError('logits must be [rows, classes] with a class at least: got {}'.format(tuple(logits.shape)))
    rows, classes = logits.shape
    k = int(k)
    if not 1 <= k <= min(MAX_K, classes):
        raise ValueError('k is {}: 1 to {} of {} classes can be listed'.format(k, min(MAX_K, classes), classes))
    logits = _rows(logits.detach())
    device = logits.device
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return top_logits(logits, k, temperature)
    values = torch.empty((rows, k), dtype=logits.dtype, device=device)
    indices = torch.empty((rows, k), dtype=torch.int32, device=device)
    rest = torch.empty((rows,), dtype=torch.float32, device=device)
    rc = _lib().pxg_top_logits(code, rows, classes, logits.data_ptr(), logits.stride(0), k, temperature, values.data_ptr(),
                               indices.data_ptr(), rest.data_ptr(), torch._C._cuda_getCurrentRawStream(device.index))
    if rc:
        _fail('pxg_top_logits', rc)
    return TopLogits(values, indices, rest, temperature)


_REDUCTIONS = ('mean', 'sum', 'none')


def _check_distill(logits, teacher, weight, reduction):
    _on_gpu('logits', logits)
    code = _floats('logits', logits)
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError('logits must be [rows, classes] with a class at least: got {}'.format(tuple(logits.shape)))
    if reduction not in _REDUCTIONS:
        raise ValueError('reduction is {!r}: one of {}'.format(reduction, ', '.join(_REDUCTIONS)))
    if not isinstance(teacher, TopLogits):
        raise TypeError('teacher must be TopLogits, not {}'.format(type(teacher).__name__))
    rows, device, t = logits.shape[0], logits.device, teacher
    for name, x in (('teacher.values', t.values), ('teacher.indices', t.indices)):
        _on_gpu(name, x, device)
    _floats('teacher.values', t.values)
    if t.indices.dtype not in (torch.int32, torch.int64):
        raise TypeError('teacher.indices is {}: int32 or int64 is needed'.format(t.indices.dtype))
    if t.values.dim() != 2 or t.values.shape[0] != rows or t.indices.shape != t.values.shape or t.values.shape[1] > MAX_K:
        raise ValueError('teacher.values and teacher.indices must be [{}, k], k up to {}: got {} and {}'.format(
            rows, MAX_K, tuple(t.values.shape), tuple(t.indices.shape)))
    if t.rest is not None:
        _f32('teacher.rest', t.rest, (rows,), device)
    if weight is not None:
        _f32('weight', weight, (rows,), device)
    for name, x in (('teacher.values', t.values), ('teacher.rest', t.rest), ('weight', weight)):
        if x is not None and x.requires_grad and torch.is_grad_enabled():
            raise ValueError('{} requires a gradient, which this loss does not give: detach it'.format(name))
    _temperature(t.temperature)
    return code


def _distill_struct(code, logits, teacher, weight, reduction):
    logits, values, indices = _rows(logits), teacher.values.contiguous(), teacher.indices.contiguous()
    s = _native.PxgDistill()
    s.struct_bytes = C.sizeof(s)
    s.dtype, s.rows, s.classes, s.row_stride = code, logits.shape[0], logits.shape[1], logits.stride(0)
    s.logits, s.k, s.value_dtype = logits.data_ptr(), values.shape[1], _DTYPES[values.dtype]
    s.values, s.indices, s.indices_are_64 = values.data_ptr(), indices.data_ptr(), int(indices.dtype == torch.int64)
    keep = [logits, values, indices]
    for name, x in (('rest', teacher.rest), ('weight', weight)):
        if x is not None:
            x = x.contiguous()
            keep.append(x)
            setattr(s, name, x.data_ptr())
    s.temperature, s.mean = teacher.temperature, int(reduction == 'mean')
    return s, keep


def _distill_forward(code, logits, teacher, weight, reduction):
    s, keep = _distill_struct(code, logits, teacher, weight, reduction)
    device, rows = logits.device, logits.shape[0]
    none = reduction == 'none'
    stats = rows * (4 + s.k)
    held = torch.empty((stats + (0 if none else rows),), dtype=torch.float32, device=device)       # stats, row_loss
    loss = torch.empty((rows,) if none else (), dtype=torch.float32, device=device)
    s.stats, s.row_loss = held.data_ptr(), loss.data_ptr() if none else held.data_ptr() + 4 * stats
    if not none:
        s.loss = loss.data_ptr()
    _call(_lib().pxg_distill_forward, s, device)
    del keep
    return loss, held


def _distill_backward(code, logits, teacher, weight, reduction, held, grad_loss):
    s, keep = _distill_struct(code, logits, teacher, weight, reduction)
    grad_loss = grad_loss.to(torch.float32).contiguous()
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    s.stats, s.grad_loss, s.grad_per_row, s.grad_logits = held.data_ptr(), grad_loss.data_ptr(), int(reduction == 'none'), grad.data_ptr()
    _call(_lib().pxg_distill_backward, s, logits.device)
    del keep
    return grad


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, code, logits, values, indices, rest, temperature, weight, reduction):
        loss, held = _distill_forward(code, logits, TopLogits(values, indices, rest, temperature), weight, reduction)
        ctx.save_for_backward(logits, values, indices, rest, weight, held)
        ctx.how = code, temperature, reduction
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        logits, values, indices, rest, weight, held = ctx.saved_tensors
        code, temperature, reduction = ctx.how
        grad = _distill_backward(code, logits, TopLogits(values, indices, rest, temperature), weight, reduction, held, grad_loss)
        return None, grad, None, None, None, None, None, None


def distillation_loss(logits, teacher, weight=None, reduction='mean'):
    """weight[n] temperature^2 KL(teacher || student) of each row, over the teacher's listed classes and one bucket for all others.

    logits [rows, classes] (or log-probabilities: a constant per row does not matter), float32, bfloat16 or float16; teacher:
    TopLogits of these rows; its temperature divides the student's logits too.  weight [rows] float32 or None; a row of weight 0
    counts for nothing whatever it holds.  reduction 'mean' (over the rows, as weighted_cross_entropy does), 'sum' or 'none'.
    float32 result, differentiable in logits.

    A class listed twice gets the sum of its shares; an index of -1 is an empty place; a row with nothing listed and no rest gives
    0; an index that is no class gives NaN, in the loss and in its row's gradient.  A student's -inf at a class that the teacher
    gives a share makes the loss inf."""
    code = _check_distill(logits, teacher, weight, reduction)
    t = teacher
    if torch.is_grad_enabled() and logits.requires_grad:
        return _differentiable(_Distillation, (logits,),
                               code, logits, t.values, t.indices, t.rest, t.temperature, weight, reduction)
    return _distill_forward(code, logits, t, weight, reduction)[0]


def distillation_loss_and_gradient(logits, teacher, weight=None, reduction='mean', grad_loss=None):
    """(loss, its gradient for the logits times grad_loss) without an autograd graph (for a captured training step).  grad_loss:
    float32, one value on the GPU, or [rows] with reduction 'none'; 1 if None."""
    code = _check_distill(logits, teacher, weight, reduction)
    shape = (logits.shape[0],) if reduction == 'none' else ()
    if grad_loss is None:
        grad_loss = torch.ones(shape, dtype=torch.float32, device=logits.device)
    else:
        _f32('grad_loss', grad_loss, shape, logits.device)
    with torch.no_grad():
        loss, held = _distill_forward(code, logits, teacher, weight, reduction)
        return loss, _distill_backward(code, logits, teacher, weight, reduction, held, grad_loss)
