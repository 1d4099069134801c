"""Operators on GPU tensors for sequence layers and their training, as hand-written HIP kernels (csrc/k_decay.hip,
csrc/k_distill.hip behind include/pxg.h).

  decay_attention        a recurrent layer whose time axis is not serial: linear attention with one decay per head, whole
                         (padded, ragged) batches, differentiable; what an LSTM layer is to ``training`` otherwise
  decay_attention_step   the same recurrence for one more step of many streams, the states updated in place
  top_logits             a teacher network's largest logits per row, with the log-sum-exp of all others
  distillation_loss      the loss of a student's logits against them, differentiable: with it the networks this package ships
                         teach others (``training.Trainer`` takes it as its ``loss_fn``)

Tensors live on one GPU; calls run on the current stream of that GPU and return without waiting.  They only launch kernels, so
they may be captured into a graph.  The library missing or a tensor on another device raises: there is no fallback.  Derivatives are
those of one backward pass: a second one and forward-mode tangents raise NotImplementedError, and so does a call that is being
recorded (torch.jit.trace, make_fx): torch sees nothing of these kernels.

Arguments are checked here; csrc/pxg_torch.cpp makes the calls and is the autograd node.
"""
import ctypes as C
import importlib.machinery
import importlib.util
import numbers
import operator
import os

import torch

from . import native as _native

__all__ = ['TopLogits', 'decay_attention', 'decay_attention_backward', 'decay_attention_step', 'distillation_loss',
           'distillation_loss_and_gradient', 'top_logits', 'MAX_WIDTH', 'MAX_K']

MAX_WIDTH = _native.PXG_DECAY_MAX_WIDTH
_MAX_PAIRS = _native.PXG_DECAY_MAX_PAIRS
MAX_K = _native.PXG_TOP_MAX_K

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)                    # enum pxg_dtype
_REDUCTIONS = {'mean': 0, 'sum': 1, 'none': 2}
_ENTRY_POINTS = ('pxg_decay_workspace_bytes', 'pxg_decay_forward', 'pxg_decay_backward', 'pxg_decay_step', 'pxg_top_logits',
                 'pxg_distill_forward', 'pxg_distill_backward')
_extension = None


# ---- checks and calls ---------------------------------------------------------------------------------------------
def _on_gpu(name, t, device=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError('{} must be a tensor, not {}'.format(name, type(t).__name__))
    if not t.is_cuda:
        raise ValueError('{} is on {}: these operators run on a GPU only'.format(name, t.device))
    if device is not None and t.device != device:
        raise ValueError('{} is on {}, the other tensors are on {}'.format(name, t.device, device))


def _floats(name, t):
    if t.dtype not in _DTYPES:
        raise TypeError('{} is {}: float32, bfloat16 or float16 is needed'.format(name, t.dtype))


def _f32(name, t, shape, device):
    _on_gpu(name, t, device)
    if t.dtype != torch.float32:
        raise TypeError('{} is {}: float32 is needed'.format(name, t.dtype))
    if tuple(t.shape) != shape:
        raise ValueError('{} has shape {}, {} is needed'.format(name, tuple(t.shape), shape))


def _ext():
    """csrc/_pxgtorch with the entry points of the loaded libpxg.so; loud when either is missing."""
    global _extension
    if _extension is None:
        lib = _native._lib or _native.load_library()
        for suffix in importlib.machinery.EXTENSION_SUFFIXES:
            path = os.path.join(_native.HERE, 'csrc', '_pxgtorch' + suffix)
            if os.path.isfile(path):
                break
        else:
            raise _native.PxgError('{} is missing: run `python -c "import __graft_entry__ as g; g.build()"`'.format(
                os.path.join(_native.HERE, 'csrc', '_pxgtorch')))
        spec = importlib.util.spec_from_file_location('_pxgtorch', path)
        extension = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(extension)
        extension.use_library([C.cast(getattr(lib, name), C.c_void_p).value for name in _ENTRY_POINTS])
        _extension = extension
    return _extension


# ---- decay attention ----------------------------------------------------------------------------------------------
def _check_decay(q, k, v, log_decay, lengths, initial_state, steps_axis=True):
    _on_gpu('q', q)
    _floats('q', q)
    device = q.device
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
    if batch * heads > _MAX_PAIRS:
        raise ValueError('{} sequences of {} heads: at most {} of both together'.format(batch, heads, _MAX_PAIRS))
    _f32('log_decay', log_decay, (heads,), device)
    if lengths is not None:
        _on_gpu('lengths', lengths, device)
        if lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError('lengths is {}: int32 or int64 is needed'.format(lengths.dtype))
        if tuple(lengths.shape) != (batch,):
            raise ValueError('lengths has shape {}, {} is needed'.format(tuple(lengths.shape), (batch,)))
    if initial_state is not None:
        _f32('initial_state', initial_state, (batch, heads, dk, dv), device)


def decay_attention(q, k, v, log_decay, lengths=None, initial_state=None, return_state=False):
    """Linear attention with one decay per head over whole sequences.

        S_t = exp(log_decay[h]) S_(t-1) + k_t v_t^T,    o_t = q_t S_t

    q, k [batch, steps, heads, dk] and v [batch, steps, heads, dv], float32, bfloat16 or float16, dk and dv of 1 to 128, any
    strides (k and v that heads share are ``expand``-ed views); log_decay [heads] float32 (-inf: no memory; one above 0
    grows, and the result is a number while exp(log_decay * steps) is one).  lengths [batch] (int32 or int64): the steps of each
    sequence, taken as 0 to steps; what lies behind them is not read, and its rows of the result are 0.
    initial_state [batch, heads, dk, dv] float32: S before the first step, 0 if None.

    Returns o [batch, steps, heads, dv] in v's type, or (o, S behind each sequence's last step, float32).  Differentiable in q,
    k, v, log_decay and initial_state.  Sums and states are held in float32 whatever the tensors' type.  Products take their
    operands in bfloat16 parts: of float32 numbers all 24 bits, less what is below 2^-24 of each term; where results are rounded to
    half precision, 16 bits of the weights exp(log_decay * (i - j)) q_i k_j inside 32 steps and of the state before them (2^-18 of
    each term).  float32 numbers of 3.38e38 and more count as infinite."""
    _check_decay(q, k, v, log_decay, lengths, initial_state)
    out, state = _ext().decay_attention(q, k, v, log_decay, lengths, initial_state, return_state)
    return (out, state) if return_state else out


def decay_attention_backward(grad_out, q, k, v, log_decay, lengths=None, initial_state=None, grad_state=None):
    """The gradients of decay_attention without an autograd graph (for a captured training step): grad_out like its result and
    grad_state like its state (or None) -> gradients of q, k, v, log_decay and initial_state (None without one)."""
    _check_decay(q, k, v, log_decay, lengths, initial_state)
    _on_gpu('grad_out', grad_out, q.device)
    if grad_out.dtype != v.dtype or grad_out.shape != v.shape:
        raise ValueError('grad_out is {} {}, v is {} {}'.format(grad_out.dtype, tuple(grad_out.shape), v.dtype, tuple(v.shape)))
    if grad_state is not None:
        _f32('grad_state', grad_state, (q.shape[0], q.shape[2], q.shape[3], v.shape[3]), q.device)
    return _ext().decay_attention_backward(grad_out, q, k, v, log_decay, lengths, initial_state, grad_state)


def decay_attention_step(q, k, v, log_decay, state, active=None):
    """One more step of many streams: q, k [batch, heads, dk], v [batch, heads, dv], state [batch, heads, dk, dv] float32,
    contiguous, updated IN PLACE.  Returns o [batch, heads, dv] in v's type.  active [batch] bool: the state of a stream that is
    not active stays as it is, and its row of the result is 0.  For inference: no gradients."""
    _check_decay(q, k, v, log_decay, None, state, steps_axis=False)
    if not state.is_contiguous():
        raise ValueError('state must be contiguous: it is updated in place')
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, log_decay, state)):
        raise RuntimeError('decay_attention_step has no gradients: call it under torch.no_grad(), or use decay_attention')
    if active is not None:
        _on_gpu('active', active, q.device)
        if active.dtype != torch.bool or tuple(active.shape) != (q.shape[0],):
            raise ValueError('active must be bool [{}]: got {} {}'.format(q.shape[0], active.dtype, tuple(active.shape)))
    return _ext().decay_step(q, k, v, log_decay, state, active)


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
        if isinstance(rows, numbers.Integral):
            if not -len(self) <= rows < len(self):
                raise IndexError('row {} of {}'.format(rows, len(self)))             # what ends a loop over the rows
            rows = slice(int(rows), int(rows) + 1 or None)
        return TopLogits(self.values[rows], self.indices[rows], None if self.rest is None else self.rest[rows], self.temperature)

    def to(self, *args, **kwargs):
        device = self.values[:0].to(*args, **kwargs).device         # moves, never casts
        return TopLogits(self.values.to(device), self.indices.to(device), None if self.rest is None else self.rest.to(device),
                         self.temperature)

    @staticmethod
    def cat(parts):
        """All rows of several answers of one temperature.  Where only some of them have a rest, the others get one of nothing
        (-inf: their listed classes are all there is)."""
        parts = list(parts)
        if not parts:
            raise ValueError('no answers to join')
        if len({p.temperature for p in parts}) != 1:
            raise ValueError('answers of different temperatures')
        rest = None
        if any(p.rest is not None for p in parts):
            rest = torch.cat([torch.full((len(p),), float('-inf'), device=p.values.device) if p.rest is None else p.rest for p in parts])
        return TopLogits(torch.cat([p.values for p in parts]), torch.cat([p.indices for p in parts]), rest, parts[0].temperature)


def _temperature(temperature):
    temperature = float(temperature)
    if not 1.2e-38 <= temperature <= 3.0e38:                       # and what float32 holds as a normal number
        raise ValueError('temperature is {}: a positive number of 1.2e-38 to 3e38 is needed'.format(temperature))
    return temperature


def top_logits(logits, k, temperature=1.0):
    """The k largest logits of each row (logits [rows, classes], k of 1 to 128) as TopLogits: descending, ties to the lowest
    class, NaN before all numbers; `rest` sums up the other classes at this temperature.  No gradients."""
    _on_gpu('logits', logits)
    _floats('logits', logits)
    temperature = _temperature(temperature)
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError('logits must be [rows, classes] with a class at least: got {}'.format(tuple(logits.shape)))
    rows, classes = logits.shape
    k = operator.index(k)
    if not 1 <= k <= min(MAX_K, classes):
        raise ValueError('k is {}: 1 to {} of {} classes can be listed'.format(k, min(MAX_K, classes), classes))
    return TopLogits(*_ext().top_logits(logits, k, temperature), temperature)


def _check_distill(logits, teacher, weight, reduction):
    _on_gpu('logits', logits)
    _floats('logits', logits)
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


def distillation_loss(logits, teacher, weight=None, reduction='mean'):
    """weight[n] temperature^2 KL(teacher || student) of each row, over the teacher's listed classes and one bucket for all others.

    logits [rows, classes] (or log-probabilities: a constant per row does not matter), float32, bfloat16 or float16; teacher:
    TopLogits of these rows; its temperature divides the student's logits too.  weight [rows] float32 or None; a row of weight 0
    counts for nothing whatever it holds.  reduction 'mean' (over the rows, as weighted_cross_entropy does), 'sum' or 'none'.
    float32 result, differentiable in logits.

    A class listed twice gets the sum of its shares; an index of -1 is an empty place; a row with nothing listed and no rest gives
    0; an index that is no class gives NaN, in the loss and in its row's gradient.  A student's -inf at a class that the teacher
    gives a share makes the loss inf."""
    _check_distill(logits, teacher, weight, reduction)
    t = teacher
    return _ext().distillation_loss(logits, t.values, t.indices, t.rest, weight, t.temperature, _REDUCTIONS[reduction])


def distillation_loss_and_gradient(logits, teacher, weight=None, reduction='mean', grad_loss=None):
    """(loss, its gradient for the logits times grad_loss) without an autograd graph (for a captured training step).  grad_loss:
    float32, one value on the GPU, or [rows] with reduction 'none'; 1 if None."""
    _check_distill(logits, teacher, weight, reduction)
    if grad_loss is not None:
        _f32('grad_loss', grad_loss, (logits.shape[0],) if reduction == 'none' else (), logits.device)
    t = teacher
    return _ext().distillation_loss_and_gradient(logits, t.values, t.indices, t.rest, weight, t.temperature, _REDUCTIONS[reduction],
                                                 grad_loss)
