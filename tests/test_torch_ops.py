"""poreplex_amd/torch_ops.py against plain 64-bit statements of the same formulas.

Tolerances.  A result of type t is rounded once: eps(t) / 2 of its value.  What is summed in float32 errs by at most
(number of roundings on the way) * 2^-24 of the sum of the ABSOLUTE terms, which the statements below compute beside the value
(`size`).  Half-precision results may also take products of operands that were split into two bfloat16 numbers: what is left over
is at most 2^-18 of each term, for the weights inside a chunk and for the state (together 2^-17)."""
import ctypes as C
import math

import numpy as np
import pytest

torch = pytest.importorskip('torch')

from poreplex_amd import native as N  # noqa: E402
from poreplex_amd import torch_ops as ops  # noqa: E402

F64 = torch.float64
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
gpu = pytest.mark.gpu


# ---- plain statements, 64 bits, on the CPU --------------------------------------------------------------------------
def recurrence(q, k, v, log_decay, lengths=None, initial_state=None):
    """(o, state), step after step."""
    b, t, h, dk = q.shape
    a = torch.exp(log_decay)[:, None, None]
    state = torch.zeros(b, h, dk, v.shape[-1], dtype=F64) if initial_state is None else initial_state
    rows = []
    for i in range(t):
        live = torch.ones(b, dtype=torch.bool) if lengths is None else i < lengths
        live = live[:, None, None, None]
        state = torch.where(live, a * state + k[:, i, :, :, None] * v[:, i, :, None, :], state)
        rows.append(torch.where(live, q[:, i, :, :, None] * state, torch.zeros((), dtype=F64)).sum(-2))
    out = torch.stack(rows, 1) if rows else torch.zeros(v.shape, dtype=F64)
    return out, state


def roundings(steps):
    """on the way of one value: the terms inside a chunk of 64 steps, the width of the states, three for each chunk passed, the
    decay factors"""
    return 64 + 128 + 3 * (steps // 64 + 1) + 64


def assert_near(got, want, size, steps, split=True, more=0.0):
    dtype = got.dtype
    tol = torch.finfo(dtype).eps / 2 * want.abs() + roundings(steps) * 2.0 ** -24 * size
    if dtype != torch.float32 and split:
        tol = tol + 2.0 ** -17 * size
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25                      # half the least step of float16
    tol = tol * (1 + 2.0 ** -7) + more + 1e-37
    off = (got.double().cpu() - want).abs()
    worst = (off - tol).max() if off.numel() else torch.tensor(-1.0)
    assert torch.isfinite(got).all() and worst <= 0, 'off by up to {:.3g}, {:.3g} over'.format(float(off.max()), float(worst))


def problem(b, t, h, dk, dv, dtype, ragged=False, state=False, seed=0, spans=(1.0, 8.0)):
    g = torch.Generator().manual_seed(seed + 7 * t + dk)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    dt = TYPES[dtype]
    p = {'q': (n(b, t, h, dk) * dk ** -0.5).to(dt), 'k': n(b, t, h, dk).to(dt), 'v': n(b, t, h, dv).to(dt)}
    p['log_decay'] = torch.log1p(-torch.exp2(-torch.linspace(*spans, h)))
    p['lengths'] = None
    if ragged:
        p['lengths'] = torch.randint(0, t + 1, (b,), generator=g)
        p['lengths'][0] = t
        if b > 1:
            p['lengths'][1] = 0
        if b > 2:
            p['lengths'][2] = min(1, t)
    p['initial_state'] = n(b, h, dk, dv) if state else None
    p['grad_out'], p['grad_state'] = n(b, t, h, dv).to(dt), n(b, h, dk, dv) if state else None
    return p


def to_f64(p):
    return {x: (y.double() if y is not None and y.is_floating_point() else y) for x, y in p.items()}


def to_gpu(p):
    return {x: (None if y is None else y.cuda()) for x, y in p.items()}


ARGS = ('q', 'k', 'v', 'log_decay', 'lengths', 'initial_state')
LEAVES = ('q', 'k', 'v', 'log_decay', 'initial_state')


def gradients(p):
    """of sum(o * grad_out) + sum(state * grad_state), through the recurrence, for every leaf."""
    p = to_f64(p)
    leaves = [p[x].clone().requires_grad_() for x in LEAVES if p[x] is not None]
    named = dict(zip([x for x in LEAVES if p[x] is not None], leaves))
    out, state = recurrence(*[named.get(x, p[x]) for x in ARGS])
    loss = (out * p['grad_out']).sum()
    if p['grad_state'] is not None:
        loss = loss + (state * p['grad_state']).sum()
    return dict(zip(named, torch.autograd.grad(loss, leaves)))


def absolute(p):
    """the same problem with every operand's absolute value: its results are the sums of the absolute terms"""
    return {x: (y.abs() if y is not None and y.is_floating_point() and x != 'log_decay' else y) for x, y in p.items()}


# (batch, steps, heads, dk, dv): one step to several chunks, chunk borders, widths that are no multiple of anything
SHAPES = [(1, 1, 1, 16, 16), (2, 5, 3, 8, 24), (3, 63, 2, 16, 16), (2, 64, 2, 32, 32), (2, 65, 1, 64, 64), (1, 130, 2, 48, 80),
          (2, 200, 1, 128, 128), (3, 100, 2, 7, 13), (2, 129, 2, 1, 1), (1, 70, 1, 33, 128), (1, 300, 4, 16, 16), (2, 67, 1, 100, 20)]


def test_plain_statement_against_differences():
    """the 64-bit gradients against central differences, along one direction for each leaf"""
    p = to_f64(problem(3, 12, 2, 4, 5, 'f32', ragged=True, state=True))
    grads = gradients(p)

    def value(q):
        out, state = recurrence(*[q[x] for x in ARGS])
        return float((out * q['grad_out']).sum() + (state * q['grad_state']).sum())
    g = torch.Generator().manual_seed(3)
    for x in LEAVES:
        d = torch.randn(p[x].shape, generator=g, dtype=F64)
        e = 1e-5
        up, down = dict(p), dict(p)
        up[x], down[x] = p[x] + e * d, p[x] - e * d
        want = float((grads[x] * d).sum())
        # third derivatives are of the size of the values, times e^2; rounding 1e-16 / e
        assert abs((value(up) - value(down)) / (2 * e) - want) < 1e-6 * (1 + abs(want)), x


@gpu
@pytest.mark.parametrize('dtype', sorted(TYPES))
@pytest.mark.parametrize('ragged,state', [(False, False), (True, True)])
@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_decay_attention(shape, ragged, state, dtype):
    p = problem(*shape, dtype, ragged, state)
    out, final = ops.decay_attention(**{x: y for x, y in to_gpu(p).items() if x in ARGS}, return_state=True)
    assert out.dtype == p['v'].dtype and final.dtype == torch.float32
    want, want_state = recurrence(*[to_f64(p)[x] for x in ARGS])
    size, size_state = recurrence(*[to_f64(absolute(p))[x] for x in ARGS])
    assert_near(out, want, size, shape[1])
    assert_near(final, want_state, size_state, shape[1])
    if ragged:
        for i, n in enumerate(p['lengths'].tolist()):
            assert (out[i, n:] == 0).all()


@gpu
@pytest.mark.parametrize('dtype', sorted(TYPES))
@pytest.mark.parametrize('ragged,state', [(False, False), (True, True)])
@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_decay_attention_gradients(shape, ragged, state, dtype):
    p = problem(*shape, dtype, ragged, state, seed=1)
    d = to_gpu(p)
    leaves = [d[x].requires_grad_() for x in LEAVES if d[x] is not None]
    out, final = ops.decay_attention(**{x: d[x] for x in ARGS}, return_state=True)
    outs, grads = ([out, final], [d['grad_out'], d['grad_state']]) if state else ([out], [d['grad_out']])
    got = dict(zip([x for x in LEAVES if d[x] is not None], torch.autograd.grad(outs, leaves, grads)))
    check_gradients(got, p, shape)
    again = ops.decay_attention_backward(d['grad_out'], *[d[x] for x in ARGS], grad_state=d['grad_state'])
    for x, y in zip(LEAVES, again):
        assert (y is None) == (x not in got) and (y is None or torch.equal(y, got[x])), x


def check_gradients(got, p, shape):
    want, size = gradients(p), gradients(absolute(p))
    assert set(got) == set(want)
    for x in got:
        # what reaches log_decay is summed over the batch and over the steps, each weighted by its distance
        n = shape[1] + (4 * shape[0] * shape[1] if x == 'log_decay' else 0)
        assert got[x].dtype == p[x].dtype and got[x].shape == p[x].shape
        assert_near(got[x], want[x], size[x].abs(), n)


@gpu
def test_decay_attention_gradients_against_differences():
    """Directional central differences of the operator's own float32 result.  With a step of e the difference errs by the result's
    rounding over 2 e and by e^2 / 6 of the third derivative along the direction, both of the size of the absolute terms."""
    p = problem(2, 150, 2, 16, 24, 'f32', ragged=True, state=True, seed=2)
    d, grads = to_gpu(p), {}
    value = lambda q: float((torch.cat([(o.double() * g.double()).flatten() for o, g in zip(  # noqa: E731
        ops.decay_attention(**{x: q[x] for x in ARGS}, return_state=True), (q['grad_out'], q['grad_state']))])).sum())
    grads = dict(zip(LEAVES, ops.decay_attention_backward(d['grad_out'], *[d[x] for x in ARGS], grad_state=d['grad_state'])))
    size = sum(float((o * g).sum()) for o, g in zip(recurrence(*[to_f64(absolute(p))[x] for x in ARGS]),
                                                    (to_f64(absolute(p))['grad_out'], to_f64(absolute(p))['grad_state'])))
    e = 2.0 ** -7
    for x in LEAVES:
        g = torch.Generator().manual_seed(5)
        direction = torch.randn(p[x].shape, generator=g).cuda()
        if x == 'log_decay':
            direction = direction.abs() * p[x].abs().cuda()               # keeps the decay below 1
        up, down = dict(d), dict(d)
        up[x], down[x] = d[x] + e * direction, d[x] - e * direction
        got, want = (value(up) - value(down)) / (2 * e), float((grads[x].double() * direction.double()).sum())
        # linear in every leaf but log_decay, where the third derivative is bounded by 27 windows' worth of the terms
        assert abs(got - want) <= roundings(150) * 2.0 ** -24 * size / e * 2 + (27 * e * e * size if x == 'log_decay' else 0), x


@gpu
@pytest.mark.parametrize('dtype', sorted(TYPES))
def test_decay_attention_layouts(dtype):
    """strides of every kind give what contiguous copies give, bit for bit: heads before steps, slices of a packed tensor (an odd
    offset: no alignment), heads that share k and v, a batch that shares q"""
    b, t, h, dk, dv = 2, 140, 3, 16, 32
    p = to_gpu(problem(b, t, h, dk, dv, dtype, True, True, seed=3))
    packed = torch.randn(b, t, h, 2 * dk + dv + 3, device='cuda').to(TYPES[dtype])
    one_k, one_v = p['k'][:, :, :1].expand(b, t, h, dk), p['v'][:, :, :1].expand(b, t, h, dv)
    variants = [
        (p['q'].transpose(1, 2).contiguous().transpose(1, 2), p['k'].permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3), p['v']),
        (packed[..., 1:1 + dk], packed[..., 1 + dk:1 + 2 * dk], packed[..., 1 + 2 * dk:1 + 2 * dk + dv]),
        (p['q'][:1].expand(b, t, h, dk), one_k, one_v),
        (p['q'].transpose(2, 3).contiguous().transpose(2, 3), p['k'], p['v']),
    ]
    go = p['grad_out'].transpose(1, 2).contiguous().transpose(1, 2)
    rest = [p['log_decay'], p['lengths'].int(), p['initial_state']]
    for q, k, v in variants:
        flat = [x.contiguous() for x in (q, k, v)]
        for x, y in zip(ops.decay_attention(q, k, v, *rest, return_state=True), ops.decay_attention(*flat, *rest, return_state=True)):
            assert torch.equal(x, y)
        for x, y in zip(ops.decay_attention_backward(go, q, k, v, *rest, grad_state=p['grad_state']),
                        ops.decay_attention_backward(p['grad_out'], *flat, *rest, grad_state=p['grad_state'])):
            assert torch.equal(x, y)
    # gradients of what the heads share are summed over them
    k1 = p['k'][:, :, :1].clone().requires_grad_()
    out = ops.decay_attention(p['q'], k1.expand(b, t, h, dk), one_v, *rest)
    shared = torch.autograd.grad(out, k1, p['grad_out'])[0]
    each = ops.decay_attention_backward(p['grad_out'], p['q'], one_k, one_v, *rest)[1]
    assert torch.allclose(shared.float(), each.sum(2, keepdim=True).float(), rtol=2 * torch.finfo(TYPES[dtype]).eps, atol=1e-6)


@gpu
@pytest.mark.parametrize('dtype', sorted(TYPES))
def test_decay_attention_padding_is_not_read(dtype):
    """NaN and inf behind the lengths change nothing, in the results or in the gradients; lengths out of range are clamped"""
    p = to_gpu(problem(4, 150, 2, 32, 16, dtype, state=True, seed=4))
    p['lengths'] = torch.tensor([150, 0, 65, 130], device='cuda')
    args = [p[x] for x in ARGS]
    want = ops.decay_attention(*args, return_state=True) + ops.decay_attention_backward(p['grad_out'], *args, grad_state=p['grad_state'])
    dirty = {x: p[x].clone() for x in ('q', 'k', 'v', 'grad_out')}
    for i, n in enumerate([150, 0, 65, 130]):
        for j, x in enumerate(dirty):
            dirty[x][i, n:] = (float('nan'), float('inf'))[(i + j) % 2]
    lengths = torch.tensor([1 << 40, -5, 65, 130], device='cuda')
    args = [dirty['q'], dirty['k'], dirty['v'], p['log_decay'], lengths, p['initial_state']]
    got = ops.decay_attention(*args, return_state=True) + ops.decay_attention_backward(dirty['grad_out'], *args, grad_state=p['grad_state'])
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    assert torch.equal(got[1][1], p['initial_state'][1]) and torch.equal(got[6][1], p['grad_state'][1])       # nothing happened there


@gpu
def test_decay_attention_is_causal_for_values_that_are_no_numbers():
    """a NaN at one step leaves every result before it as it was"""
    p = to_gpu(problem(1, 200, 1, 16, 16, 'f32', seed=5))
    want = ops.decay_attention(p['q'], p['k'], p['v'], p['log_decay'])
    for name in ('k', 'v', 'q'):
        bad = dict(p)
        bad[name] = p[name].clone()
        bad[name][0, 101, 0, 3] = float('nan')
        got = ops.decay_attention(bad['q'], bad['k'], bad['v'], p['log_decay'])
        assert torch.equal(got[0, :101], want[0, :101]) and torch.isnan(got[0, 101]).any()


@gpu
def test_decay_attention_extreme_decays():
    """no memory at all (-inf), no decay (0), a decay that underflows within a few steps"""
    p = problem(2, 190, 3, 16, 16, 'f32', ragged=True, state=True, seed=6)
    p['log_decay'] = torch.tensor([-math.inf, 0.0, -40.0])
    d = to_gpu(p)
    got = ops.decay_attention(**{x: d[x] for x in ARGS}, return_state=True)
    want = recurrence(*[to_f64(p)[x] for x in ARGS])
    size = recurrence(*[to_f64(absolute(p))[x] for x in ARGS])
    for x, y, z in zip(got, want, size):
        assert_near(x, y, z, 190)
    grads = ops.decay_attention_backward(d['grad_out'], *[d[x] for x in ARGS], grad_state=d['grad_state'])
    assert all(torch.isfinite(x).all() for x in grads) and grads[3][0] == 0
    p['log_decay'] = torch.tensor([-200.0, 0.0, -40.0])            # exp(-200) is 0 in 32 bits; its gradients are finite in 64
    check_gradients(dict(zip(LEAVES, grads)), p, (2, 190, 3, 16, 16))


@gpu
@pytest.mark.parametrize('dtype', sorted(TYPES))
@pytest.mark.parametrize('state', [False, True])
@pytest.mark.parametrize('steps', [1, 2, 17, 30, 33, 70, 700])
def test_decay_attention_growing_decays(steps, state, dtype):
    """log_decay above 0: numbers as long as exp(log_decay * steps) is one, however short the sequences are"""
    p = problem(5, steps, 3, 16, 24, dtype, True, state, seed=40)
    # (the gradient of log_decay is `steps` times a sum of such factors; float16 results end at 65 504, without a state and with
    # one step they do not depend on the decay)
    most = 3.0 if dtype == 'f16' and (state or steps > 1) else 60.0
    p['log_decay'] = torch.tensor([most / steps, 0.5 / steps, -0.1])
    d = to_gpu(p)
    got = ops.decay_attention(**{x: d[x] for x in ARGS}, return_state=True)
    want = recurrence(*[to_f64(p)[x] for x in ARGS])
    size = recurrence(*[to_f64(absolute(p))[x] for x in ARGS])
    for x, y, z in zip(got, want, size):
        assert_near(x, y, z, steps)
    grads = ops.decay_attention_backward(d['grad_out'], *[d[x] for x in ARGS], grad_state=d['grad_state'])
    check_gradients({x: y for x, y in zip(LEAVES, grads) if y is not None}, p, (5, steps, 3, 16, 24))


@gpu
def test_decay_attention_empty_and_long():
    for b, t in ((0, 5), (2, 0)):
        p = to_gpu(problem(max(b, 1), max(t, 1), 2, 8, 8, 'f32', state=True))
        cut = {x: (p[x][:b] if p[x] is not None and x != 'log_decay' else p[x]) for x in p}
        cut.update({x: cut[x][:, :t] for x in ('q', 'k', 'v', 'grad_out')})
        out, state = ops.decay_attention(**{x: cut[x] for x in ARGS}, return_state=True)
        assert out.shape == (b, t, 2, 8) and torch.equal(state, cut['initial_state'])
        grads = ops.decay_attention_backward(cut['grad_out'], *[cut[x] for x in ARGS], grad_state=cut['grad_state'])
        assert torch.equal(grads[4], cut['grad_state']) and (grads[3] == 0).all()
    # one long row, and its continuation from a state is the same row
    p = to_gpu(problem(1, 9001, 2, 16, 16, 'f32', state=True, seed=8))
    whole, state = ops.decay_attention(**{x: p[x] for x in ARGS}, return_state=True)
    cpu = problem(1, 9001, 2, 16, 16, 'f32', state=True, seed=8)
    want = recurrence(*[to_f64(cpu)[x] for x in ARGS])
    size = recurrence(*[to_f64(absolute(cpu))[x] for x in ARGS])
    assert_near(whole, want[0], size[0], 9001)
    assert_near(state, want[1], size[1], 9001)
    cut = 4321
    first, middle = ops.decay_attention(p['q'][:, :cut], p['k'][:, :cut], p['v'][:, :cut], p['log_decay'], None, p['initial_state'], True)
    second, last = ops.decay_attention(p['q'][:, cut:], p['k'][:, cut:], p['v'][:, cut:], p['log_decay'], None, middle, True)
    assert_near(torch.cat([first, second], 1), want[0], size[0], 9001)
    assert_near(last, want[1], size[1], 9001)
    got = dict(zip(LEAVES, ops.decay_attention_backward(p['grad_out'], *[p[x] for x in ARGS], grad_state=p['grad_state'])))
    check_gradients(got, cpu, (1, 9001, 2, 16, 16))


# ---- one step ---------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize('dtype', sorted(TYPES))
@pytest.mark.parametrize('shape', [(1, 1, 16, 16), (5, 4, 64, 64), (3, 2, 7, 13), (2, 3, 128, 128), (70, 2, 48, 40), (2, 1, 1, 1),
                                   (4, 2, 33, 100)], ids=str)
def test_decay_attention_step(shape, dtype):
    b, h, dk, dv = shape
    p = problem(b, 1, h, dk, dv, dtype, state=True, seed=9)
    d = to_gpu(p)
    state = d['initial_state'].clone()
    active = torch.arange(b, device='cuda') % 3 != 1
    out = ops.decay_attention_step(d['q'][:, 0], d['k'][:, 0], d['v'][:, 0], d['log_decay'], state, active=active)
    want, want_state = recurrence(*[to_f64(p)[x] for x in ARGS])
    size, size_state = recurrence(*[to_f64(absolute(p))[x] for x in ARGS])
    on = active.cpu()
    assert_near(out[active], want[:, 0][on], size[:, 0][on], 1)
    assert_near(state[active], want_state[on], size_state[on], 1)
    assert (out[~active] == 0).all() and torch.equal(state[~active], d['initial_state'][~active])


@gpu
def test_steps_are_the_sequence():
    p = to_gpu(problem(3, 90, 2, 32, 48, 'f32', state=True, seed=10))
    state, rows = p['initial_state'].clone(), []
    for i in range(90):
        rows.append(ops.decay_attention_step(p['q'][:, i], p['k'][:, i], p['v'][:, i], p['log_decay'], state))
    out, final = ops.decay_attention(**{x: p[x] for x in ARGS}, return_state=True)
    cpu = problem(3, 90, 2, 32, 48, 'f32', state=True, seed=10)
    size = recurrence(*[to_f64(absolute(cpu))[x] for x in ARGS])
    assert_near(torch.stack(rows, 1), out.double().cpu(), 2 * size[0], 90)
    assert_near(state, final.double().cpu(), 2 * size[1], 90)


# ---- a teacher's top logits ---------------------------------------------------------------------------------------------
def top_statement(x, k, temperature):
    indices = np.stack([sorted(range(x.shape[1]), key=lambda v: (not math.isnan(row[v]), -row[v] if not math.isnan(row[v]) else 0, v))[:k]
                        for row in x])
    rest = np.empty(len(x))
    for i, row in enumerate(x):
        left = np.delete(row, indices[i])
        most = left.max() if len(left) else -math.inf
        rest[i] = most if math.isinf(most) else most / temperature + math.log(np.exp((left - most) / temperature).sum())
    return np.take_along_axis(x, indices, 1), indices, rest


@gpu
@pytest.mark.parametrize('dtype', sorted(TYPES))
@pytest.mark.parametrize('rows,classes,k', [(1, 1, 1), (7, 5, 3), (4, 5, 5), (3, 128, 128), (3, 129, 128), (5, 257, 4), (2, 1000, 100),
                                            (3, 5003, 31), (2, 20011, 128), (1, 70001, 64)])
def test_top_logits(rows, classes, k, dtype):
    g = torch.Generator().manual_seed(classes + k)
    x = (torch.randn(rows, classes, generator=g) * 3).to(TYPES[dtype])
    x[-1] = torch.randint(0, 3, (classes,), generator=g).to(TYPES[dtype])            # ties everywhere
    check_top(x, k, 2.0)


def check_top(x, k, temperature):
    t = ops.top_logits(x.cuda(), k, temperature)
    values, indices, rest = top_statement(x.double().numpy(), k, temperature)
    assert t.values.dtype == x.dtype and t.indices.dtype == torch.int32 and t.rest.dtype == torch.float32
    assert np.array_equal(t.indices.cpu().numpy(), indices)
    assert np.array_equal(t.values.double().cpu().numpy(), values, equal_nan=True)
    got = t.rest.double().cpu().numpy()
    fine = np.isfinite(rest)
    assert np.array_equal(got[~fine], rest[~fine], equal_nan=True)
    # each exponential errs by 4 roundings and its exponent's own, of at most 2^-24 of |x|; the sum by its depth; the result by half a step
    tol = 2.0 ** -24 * (np.abs(rest[fine]) + 64 + 2 * np.abs(np.nan_to_num(x.double().numpy(), posinf=0, neginf=0)).max() / temperature)
    off = np.abs(got[fine] - rest[fine])
    assert (off <= tol).all(), off.max()


@gpu
@pytest.mark.parametrize('dtype', sorted(TYPES))
@pytest.mark.parametrize('rows,classes,k', [(1, 2, 1), (33, 8, 8), (65, 9, 4), (17, 16, 1), (9, 17, 17), (5, 32, 31), (7, 33, 3), (6, 64, 64),
                                            (6, 65, 64)])
def test_top_logits_of_few_classes(rows, classes, k, dtype):
    g = torch.Generator().manual_seed(classes + k)
    x = (torch.randn(rows, classes + 3, generator=g) * 3).to(TYPES[dtype])
    x[-1] = torch.randint(0, 3, (classes + 3,), generator=g).to(TYPES[dtype])
    check_top(x[:, :classes].contiguous(), k, 1.5)
    t, u = ops.top_logits(x.cuda()[:, 2:-1], k, 1.5), ops.top_logits(x[:, 2:-1].contiguous().cuda(), k, 1.5)     # not aligned
    for name in ('values', 'indices', 'rest'):
        assert torch.equal(getattr(t, name), getattr(u, name))


@gpu
def test_top_logits_strange_rows_of_few_classes():
    inf, nan = math.inf, math.nan
    for classes in (5, 40):
        x = torch.zeros(9, classes)
        x[0] = -inf
        x[1, 2:] = -inf
        x[2, 3] = inf
        x[3, 1:] = inf
        x[4, 4] = nan
        x[5] = torch.arange(float(classes))
        x[6, :4] = nan
        x[7, ::2] = -0.0
        x[8] = torch.finfo(torch.float32).min
        for k in (1, 2, 5):
            check_top(x, k, 1.0)


@gpu
def test_top_logits_strange_rows():
    inf, nan = math.inf, math.nan
    x = torch.zeros(9, 300)
    x[0] = -inf
    x[1, 5:] = -inf
    x[2, 7] = inf
    x[3, 100:110] = inf
    x[4, 200] = nan
    x[5] = torch.arange(300.0)
    x[6] = -torch.arange(300.0)
    x[7, ::2] = -0.0
    x[8] = torch.finfo(torch.float32).min
    for k in (1, 4, 8, 128):
        check_top(x, k, 1.0)
    # a row of one value, longer than any buffer; a row whose largest lie behind one another
    check_top(torch.ones(2, 40000), 128, 1.0)
    check_top(torch.arange(40000.0).repeat(2, 1), 128, 1.0)
    check_top((torch.arange(40000) // 64 % 7).float().repeat(2, 1), 100, 1.0)
    # rows of a wider tensor, not aligned
    wide = torch.randn(6, 1001)
    t, u = ops.top_logits(wide.cuda()[:, 1:], 10), ops.top_logits(wide[:, 1:].contiguous().cuda(), 10)
    assert torch.equal(t.indices, u.indices) and torch.equal(t.rest, u.rest)
    assert len(ops.top_logits(torch.empty(0, 7, device='cuda'), 3)) == 0


# ---- the distillation loss ----------------------------------------------------------------------------------------------
def distill_statement(x, values, indices, rest, temperature, weight=None):
    """(row losses, gradient of their sum), 64 bits, one row after the other"""
    n, classes = x.shape
    loss, grad, size = np.zeros(n), np.zeros_like(x), np.zeros(n)
    for r in range(n):
        w = 1.0 if weight is None else weight[r]
        at = {}
        t = [(v / temperature, i) for v, i in zip(values[r], indices[r]) if i != -1]
        tail = -math.inf if rest is None else rest[r]
        most = max([v for v, _ in t] + [tail])
        if w == 0 or most == -math.inf:
            continue
        total = sum(math.exp(v - most) for v, _ in t) + math.exp(tail - most)
        for v, i in t:
            at[i] = at.get(i, 0.0) + math.exp(v - most) / total
        pr = math.exp(tail - most) / total
        y = x[r] / temperature
        z = y.max() + math.log(np.exp(y - y.max()).sum())
        q = np.exp(y - z)
        off = np.ones(classes, bool)
        off[list(at)] = False
        qr = q[off].sum()
        terms = [p * (math.log(p) - (y[i] - z)) for i, p in at.items() if p > 0] + ([pr * (math.log(pr) - math.log(qr))] if pr > 0 else [])
        loss[r] = w * temperature ** 2 * sum(terms)
        g = q.copy()
        if pr > 0:
            g[off] -= pr * q[off] / qr
        for i, p in at.items():
            g[i] -= p
        grad[r] = w * temperature * g
        # what float32 puts in: the largest exponent's rounding in each share
        size[r] = w * temperature ** 2 * (1 + np.abs(y[np.isfinite(y)] - y.max()).max())
    return loss, grad, size


def distill_problem(rows, classes, k, dtype, temperature, seed=0):
    g = torch.Generator().manual_seed(classes * 3 + k + seed)
    teacher = torch.randn(rows, classes, generator=g) * 3
    x = (teacher + torch.randn(rows, classes, generator=g)).to(TYPES[dtype])
    values, indices, rest = top_statement(teacher.to(TYPES[dtype]).double().numpy(), k, temperature)
    weight = torch.rand(rows, generator=g)
    weight[rows // 2] = 0.0
    return x, ops.TopLogits(torch.from_numpy(values).to(TYPES[dtype]), torch.from_numpy(indices).int(), torch.from_numpy(rest).float(),
                            temperature), weight


def check_distill(x, teacher, weight, reduction='none', grad_loss=None):
    rows = len(x)
    d, w = x.cuda().requires_grad_(), None if weight is None else weight.cuda()
    t = teacher.to('cuda')
    loss = ops.distillation_loss(d, t, w, reduction)
    g = torch.linspace(0.5, 1.5, rows) if reduction == 'none' else torch.tensor(1.25)
    grad = torch.autograd.grad(loss, d, g.cuda())[0]
    both = ops.distillation_loss_and_gradient(d, t, w, reduction, g.cuda())
    assert torch.equal(both[0], loss.detach()) and torch.equal(both[1], grad)
    want, want_grad, size = distill_statement(x.double().numpy(), teacher.values.double().numpy(), teacher.indices.numpy(),
                                              None if teacher.rest is None else teacher.rest.double().numpy(), teacher.temperature,
                                              None if weight is None else weight.double().numpy())
    scale = g.double().numpy() if reduction == 'none' else np.full(rows, float(g) / (rows if reduction == 'mean' else 1))
    want_grad = want_grad * scale[:, None]
    if reduction != 'none':
        want, size = want.sum() / (rows if reduction == 'mean' else 1), size.sum() / (rows if reduction == 'mean' else 1)
    # a share errs by the roundings of an exponential (its exponent's are in `size`) and of a sum over the classes
    assert loss.dtype == torch.float32 and grad.dtype == x.dtype
    off = np.abs(loss.detach().double().cpu().numpy() - want)
    assert (off <= 2.0 ** -24 * (np.abs(want) + 64 * size)).all(), (off.max(), np.max(size))
    room = (np.abs(scale) * (1.0 if weight is None else weight.double().numpy()) * teacher.temperature)[:, None]
    per = 2.0 ** -24 * 64 * (1 + np.abs(np.nan_to_num(x.double().numpy(), neginf=0.0)).max(1, keepdims=True) / teacher.temperature) * room
    q = torch.softmax(x.double() / teacher.temperature, 1).numpy()
    # an unlisted class's gradient is a multiple of its share; a listed one's a difference of two shares
    bound = per * np.maximum(q, np.where(np.abs(want_grad) > 0, 2.0 ** -24, 0))
    for r in range(rows):
        bound[r, teacher.indices[r].clamp(min=0).numpy()] = per[r]
    if x.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    tol = torch.finfo(x.dtype).eps / 2 * np.abs(want_grad) + bound + 1e-37
    off = np.abs(grad.double().cpu().numpy() - want_grad)
    assert (off <= tol * (1 + 2.0 ** -7)).all(), ((off - tol).max(), off.max())
    return loss, grad


@gpu
@pytest.mark.parametrize('dtype', sorted(TYPES))
@pytest.mark.parametrize('rows,classes,k,temperature', [(1, 1, 1, 1.0), (6, 5, 3, 2.0), (5, 5, 5, 1.5), (4, 300, 1, 1.0), (3, 257, 128, 4.0),
                                                        (3, 2048, 17, 1.0), (5, 5001, 100, 4.0), (2, 40003, 64, 1.0)])
def test_distillation_loss(rows, classes, k, temperature, dtype):
    x, teacher, weight = distill_problem(rows, classes, k, dtype, temperature)
    for reduction in ('none', 'mean', 'sum'):
        check_distill(x, teacher, weight, reduction)
    check_distill(x, teacher, None)
    check_distill(x, ops.TopLogits(teacher.values, teacher.indices.long(), None, temperature), weight)


@gpu
def test_distillation_loss_against_differences():
    """of the operator's own loss: an error of the loss's rounding over the step, and a step's square times the third derivative,
    which is below w / temperature^3 * temperature^2 per unit of the direction's cube"""
    x, teacher, weight = distill_problem(4, 200, 9, 'f32', 2.0, seed=1)
    t, w = teacher.to('cuda'), weight.cuda()
    loss, grad = ops.distillation_loss_and_gradient(x.cuda(), t, w, 'sum')
    g = torch.Generator().manual_seed(2)
    for _ in range(3):
        d = torch.randn(x.shape, generator=g).cuda()
        e = 2.0 ** -6
        up, down = (ops.distillation_loss(x.cuda() + s * e * d, t, w, 'sum').double() for s in (1, -1))
        want = float((grad.double() * d.double()).sum())
        room = 64 * 16 * 4 * float(weight.sum()) * 2.0 ** -24 / e + e * e * float(weight.sum()) * float(d.abs().max()) ** 3
        assert abs(float(up - down) / (2 * e) - want) <= room


@gpu
def test_distillation_loss_strange_rows():
    inf, nan = math.inf, math.nan
    x, teacher, _ = distill_problem(12, 50, 6, 'f32', 1.0, seed=3)
    v, i, r = teacher.values, teacher.indices, teacher.rest
    i[1, 2:] = -1                                        # empty places
    i[2] = -1                                            # nothing listed: the rest alone
    i[3, 4] = i[3, 1]                                    # a class twice
    i[4] = i[4, 0]                                       # one class in every place
    v[5, 3:] = -inf                                      # places without a share
    r[6] = -inf                                          # nothing unlisted
    i[7], r[7] = -1, -inf                                # nothing at all
    x[8, i[8, 5].item()] -= 200.0                        # far below, but a number
    x[9, [c for c in range(50) if c not in i[9].tolist()]] = -150.0           # the unlisted far below the listed
    weight = torch.ones(12)
    weight[10] = 0.0
    x[10] = nan                                          # a row that does not count may hold anything
    x[11, [c for c in range(50) if c not in i[11].tolist()][3]] = -inf        # one class ruled out
    rows = list(range(12))
    rows.remove(10)
    loss, grad = check_distill(x[rows], teacher[rows], None)
    assert float(loss[7].detach()) == 0 and (grad[7] == 0).all()
    loss, grad = ops.distillation_loss_and_gradient(x.cuda(), teacher.to('cuda'), weight.cuda(), 'none')
    assert float(loss[10]) == 0 and (grad[10] == 0).all() and torch.isfinite(loss).all() and torch.isfinite(grad).all()
    # a share where the student has none: infinite, with finite gradients; what is no class: NaN in its row alone
    x, teacher, _ = distill_problem(4, 50, 6, 'f32', 1.0, seed=4)
    x[1, int(teacher.indices[1, 0])] = -inf
    teacher.indices[2, 1], teacher.indices[3, 0] = 50, -2
    loss, grad = ops.distillation_loss_and_gradient(x.cuda(), teacher.to('cuda'), None, 'none')
    assert math.isinf(loss[1]) and torch.isfinite(grad[:2]).all() and torch.isfinite(loss[0])
    assert torch.isnan(loss[2:]).all() and torch.isnan(grad[2:]).all()
    assert torch.isnan(ops.distillation_loss(x.cuda(), teacher.to('cuda')))
    empty = ops.TopLogits(torch.empty(0, 3, device='cuda'), torch.empty(0, 3, dtype=torch.int32, device='cuda'))
    none = torch.empty(0, 9, device='cuda', requires_grad=True)
    assert float(ops.distillation_loss(none.detach(), empty, reduction='sum')) == 0


# ---- together, streams, graphs ----------------------------------------------------------------------------------------------
@gpu
def test_teacher_student_together():
    """a layer's result through a linear map is the student, another map the teacher: one step's loss and gradients"""
    g = torch.Generator().manual_seed(11)
    b, t, h, d, classes, k, tau = 6, 70, 2, 16, 37, 5, 2.0
    p = problem(b, t, h, d, d, 'f32', ragged=True, seed=11)
    p['lengths'][1] = 3
    head, teach = torch.randn(h * d, classes, generator=g) * 0.3, torch.randn(b * t, classes, generator=g) * 2
    weight = (torch.arange(t) < p['lengths'][:, None]).float().flatten()
    teacher = ops.top_logits(teach.cuda(), k, tau)
    leaf = [p[x].cuda().requires_grad_() for x in ('q', 'k', 'v', 'log_decay')] + [head.cuda().requires_grad_()]
    out = ops.decay_attention(*leaf[:4], lengths=p['lengths'].cuda())
    loss = ops.distillation_loss(out.reshape(b * t, h * d) @ leaf[4], teacher, weight.cuda())
    got = torch.autograd.grad(loss, leaf)
    plain = [x.detach().double().cpu().requires_grad_() for x in leaf]
    o, _ = recurrence(*plain[:4], p['lengths'])
    y = o.reshape(b * t, h * d) @ plain[4] / tau
    values, indices, rest = top_statement(teach.double().numpy(), k, tau)
    both = torch.log_softmax(torch.cat([torch.from_numpy(values) / tau, torch.from_numpy(rest)[:, None]], 1), 1)
    z, index = torch.log_softmax(y, 1), torch.from_numpy(indices)
    away = torch.ones_like(z, dtype=torch.bool).scatter_(1, index, False)
    logq = torch.cat([z.gather(1, index), z.masked_fill(~away, -math.inf).logsumexp(1, keepdim=True)], 1)
    want_loss = (weight.double() * (both.exp() * (both - logq)).sum(1)).mean() * tau ** 2
    want = torch.autograd.grad(want_loss, plain)
    # a float32 product of 32 terms and sums of up to 420 rows on the way: 1e-5 of the gradient's norm is 2^-24 * 168
    assert abs(loss.item() - want_loss.item()) <= 1e-5 * abs(want_loss.item())
    for x, y in zip(got, want):
        assert float((x.double().cpu() - y).norm()) <= 1e-5 * float(y.norm())


@gpu
def test_streams_and_graphs():
    """another stream than the tensors' own; every call captured (two graphs, alive together) and replayed several times with
    eager work between, new inputs each time"""
    p = to_gpu(problem(2, 200, 2, 32, 32, 'bf16', True, True, seed=12))
    x, teacher, weight = distill_problem(33, 700, 9, 'f32', 2.0, seed=12)
    x, teacher, weight = x.cuda(), teacher.to('cuda'), weight.cuda()
    args = [p[n] for n in ARGS]
    state = p['initial_state'].clone()

    def everything():
        outs = list(ops.decay_attention(*args, return_state=True))
        outs += ops.decay_attention_backward(p['grad_out'], *args, grad_state=p['grad_state'])
        outs.append(ops.decay_attention_step(p['q'][:, 0], p['k'][:, 0], p['v'][:, 0], p['log_decay'], state))
        t = ops.top_logits(x, 9, 2.0)
        outs += [t.values, t.indices, t.rest, *ops.distillation_loss_and_gradient(x, teacher, weight)]
        return outs + [state]
    first = state.clone()
    want = [y.clone() for y in everything()]
    state.copy_(first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [y.clone() for y in everything()]
    torch.cuda.current_stream().wait_stream(side)
    for y, z in zip(got, want):
        assert torch.equal(y, z)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = everything()
        graphs.append((graph, outs))
    for turn in range(4):
        p['q'].mul_(0.5), x.add_(torch.randn_like(x))
        state.copy_(first)
        want = [y.clone() for y in everything()]
        for graph, outs in graphs:
            state.copy_(first)
            graph.replay()
            torch.cuda.synchronize()
            for y, z in zip(outs, want):
                assert torch.equal(y, z), turn


@gpu
def test_captured_backward_beside_an_eager_graph():
    """Refused before anything happens: the backward pass would have to wait, inside the capture, for the stream of the eager
    graph.  With that graph gone the same capture works."""
    p = to_gpu(problem(1, 20, 1, 8, 8, 'f32', seed=13))
    q = p['q'].requires_grad_()
    eager = ops.decay_attention(q, p['k'], p['v'], p['log_decay'])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='alive'):
        with torch.cuda.graph(graph):
            ops.decay_attention(q, p['k'], p['v'], p['log_decay'])
    torch.cuda.synchronize()
    want = torch.autograd.grad(eager, q, p['grad_out'])[0]
    del eager, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(ops.decay_attention(q, p['k'], p['v'], p['log_decay']), q, p['grad_out'])[0]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize('rows,classes,k,dtype', [(2050, 5003, 31, 'f32'), (2048, 5001, 32, 'bf16'), (4097, 1031, 1, 'f16'),
                                                  (1100, 3001, 64, 'f32'), (1030, 1200, 50, 'f16'), (1025, 33001, 20, 'bf16')])
def test_top_logits_of_many_rows(rows, classes, k, dtype):
    """a wave or two for each row, however long"""
    inf, nan = math.inf, math.nan
    g = torch.Generator().manual_seed(classes)
    x = torch.randn(rows, classes, generator=g) * 3
    x[0], x[1], x[2] = -inf, torch.arange(float(classes)), -torch.arange(float(classes))
    x[3, 5:] = -inf
    x[4, 7], x[5, 100:140], x[6, 900], x[7] = inf, inf, nan, 1.0
    x[8] = torch.arange(classes) // 64 % 7
    x[9] = torch.finfo(TYPES[dtype]).min
    x[10, 3:40] = nan
    x[-1] = torch.randint(0, 3, (classes,), generator=g).float()
    check_top(x.to(TYPES[dtype]), k, 1.0)


def masked_rows(rows, classes, k, dtype, seed=46):
    """rows of numbers where a mask leaves none to all of them, in one piece, scattered, or at the places of one thread"""
    g = torch.Generator().manual_seed(seed + classes)
    low = torch.finfo(TYPES[dtype]).min
    x, r = torch.full((rows, classes), -math.inf), 0
    for count in sorted({min(c, classes) for c in (0, 1, 2, k - 1, k, k + 1, 130, 500, 2000, 5000)}):
        places = [torch.arange(count), classes - count + torch.arange(count), (classes - count) // 2 + torch.arange(count),
                  torch.randperm(classes, generator=g)[:count], (torch.arange(count) * 4096) % classes + torch.arange(count) * 4096 // classes]
        for at in places:
            at = at.unique().clamp(max=classes - 1)
            x[r, :] = -math.inf if r % 2 else low                   # the type's lowest number masks as well, and is a number
            x[r, at] = torch.randn(len(at), generator=g) * 3
            r += 1
    x[r] = low
    x[r + 1, classes // 2:] = low                                   # both kinds
    x[r + 2, :classes // 2] = low
    x[r + 3, 1::2], x[r + 3, 4] = low, 1.0
    x[r + 4, classes // 3], x[r + 4, classes - 1] = math.inf, math.nan
    x[r + 5, -3:] = low
    x[r + 6:] = torch.randn(rows - r - 6, classes, generator=g)
    x[r + 6:, :classes // 2] = -math.inf
    return x.to(TYPES[dtype])


@gpu
@pytest.mark.parametrize('rows,classes,k,dtype', [(60, 700, 9, 'f32'), (60, 5003, 128, 'bf16'), (70, 30001, 100, 'bf16'), (80, 40000, 128, 'f32'),
                                                  (1100, 3001, 64, 'f32'), (1100, 9001, 50, 'f16'), (2050, 5003, 31, 'f32'),
                                                  (2050, 3001, 1, 'f16')])
def test_top_logits_of_masked_rows(rows, classes, k, dtype):
    x = masked_rows(rows, classes, k, dtype)
    check_top(x, k, 1.0)
    # the rest of each row by what its own numbers allow (check_top goes by the largest of all): masked places add nothing beside
    # others, and count one each where they are all that is left
    got, rest = ops.top_logits(x.cuda(), k, 1.0).rest.double().cpu().numpy(), top_statement(x.double().numpy(), k, 1.0)[2]
    for r in range(rows):
        if np.isfinite(rest[r]):
            own = x[r][torch.isfinite(x[r]) & (x[r] > torch.finfo(x.dtype).min)].double().abs()
            most = float(own.max()) if len(own) else 0.0
            assert abs(got[r] - rest[r]) <= 2.0 ** -24 * (abs(rest[r]) + 64 + 2 * most), r


@gpu
@pytest.mark.parametrize('rows,classes,k,dtype', [(2047, 50001, 64, 'bf16'), (500, 131071, 100, 'f32'), (4096, 8000, 8, 'f16'), (100, 60001, 128, 'bf16')])
def test_masked_rows_take_one_pass(rows, classes, k, dtype):
    """masks that leave a few, a thousand or half of the classes: not ten times the work (bisection takes thirty)"""
    x = torch.randn(rows, classes, device='cuda', generator=torch.Generator('cuda').manual_seed(47)).to(TYPES[dtype])

    def time_of(x):
        ops.top_logits(x, k)
        times = []
        for _ in range(5):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            for _ in range(5):
                ops.top_logits(x, k)
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end) / 5)
        return min(times)
    free = time_of(x)
    for mask in (-math.inf, torch.finfo(x.dtype).min):
        for keep in (slice(0, 40), slice(classes // 3, classes // 3 + 1000), slice(classes // 2, classes)):
            masked = torch.full_like(x, mask)
            masked[:, keep] = x[:, keep]
            assert time_of(masked) < 8 * free, (mask, keep)


@gpu
@pytest.mark.parametrize('rows,classes,k,dtype', [(4096, 2047, 5, 'f32'), (4099, 1500, 100, 'bf16')])
def test_distillation_loss_of_many_rows(rows, classes, k, dtype):
    """a wave for each row, against a workgroup for each row of a part of them: both within a few roundings of float32 of the same
    loss, and of gradients that are rounded to their type"""
    x, teacher, weight = distill_problem(rows, classes, k, dtype, 2.0, seed=30)
    x, teacher, weight = x.cuda(), teacher.to('cuda'), weight.cuda()
    loss, grad = ops.distillation_loss_and_gradient(x, teacher, weight, 'none')
    for part in (slice(0, 700), slice(rows - 700, rows)):
        one, g = ops.distillation_loss_and_gradient(x[part], teacher[part], weight[part], 'none')
        assert torch.allclose(loss[part], one, rtol=1e-5, atol=1e-5 * float(one.abs().max()))
        assert torch.allclose(grad[part].float(), g.float(), rtol=1e-5 + torch.finfo(g.dtype).eps, atol=1e-6 * float(g.float().abs().max()))
    want, gradient = distill_statement(*[y.double().cpu().numpy() for y in (x[-40:], teacher.values[-40:])],
                                       teacher.indices[-40:].cpu().numpy(), None if teacher.rest is None else teacher.rest[-40:].double().cpu().numpy(),
                                       2.0, weight[-40:].double().cpu().numpy())[:2]
    assert np.allclose(loss[-40:].double().cpu().numpy(), want, rtol=1e-4, atol=1e-4 * np.abs(want).max())
    assert np.allclose(grad[-40:].double().cpu().numpy(), gradient, rtol=1e-4 + torch.finfo(grad.dtype).eps, atol=1e-4 * np.abs(gradient).max())


# ---- calls that are allowed and unusual ---------------------------------------------------------------------------------
@gpu
def test_captured_backward_of_what_a_leaf_was_made_into():
    """the leaf behind a view, a cast or a layer counts as well"""
    p = to_gpu(problem(1, 20, 1, 8, 8, 'f32', seed=14))
    leaf = p['q'].requires_grad_()
    call = lambda: ops.decay_attention(leaf * 2, p['k'], p['v'], p['log_decay'])                   # noqa: E731
    eager = call()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='alive'):
        with torch.cuda.graph(graph):
            call()
    torch.cuda.synchronize()
    want = torch.autograd.grad(eager, leaf, p['grad_out'])[0]
    x, teacher, weight = distill_problem(3, 70, 9, 'f32', 2.0, seed=14)
    x, teacher, weight = x.cuda().requires_grad_(), teacher.to('cuda'), weight.cuda()
    eager = ops.distillation_loss(x.view(3, 70), teacher, weight)
    with pytest.raises(RuntimeError, match='alive'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.distillation_loss(x.view(3, 70), teacher, weight)
    torch.cuda.synchronize()
    del eager, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(call(), leaf, p['grad_out'])[0]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@gpu
def test_what_autograd_refuses():
    p = to_gpu(problem(2, 20, 1, 8, 8, 'f32', False, True, seed=15))
    args = [p[n] for n in ARGS]
    args[0].requires_grad_()
    out = ops.decay_attention(*args)
    with pytest.raises(NotImplementedError, match='second derivative'):
        torch.autograd.grad(out.sum(), args[0], create_graph=True)
    out = ops.decay_attention(*args)
    args[1].add_(1.0)                                              # k is needed as it was
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.sum().backward()
    x, teacher, weight = distill_problem(3, 7, 2, 'f32', 2.0, seed=15)
    x, teacher, weight = x.cuda().requires_grad_(), teacher.to('cuda'), weight.cuda()
    with pytest.raises(NotImplementedError, match='second derivative'):
        torch.autograd.grad(ops.distillation_loss(x, teacher, weight), x, create_graph=True)
    loss = ops.distillation_loss(x, teacher, weight)
    teacher.indices.zero_()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


@gpu
def test_inference_mode_and_twice_backward():
    with torch.inference_mode():
        p = to_gpu(problem(2, 3, 2, 16, 8, 'bf16', False, True, seed=16))
        whole, last = ops.decay_attention(*[p[n] for n in ARGS], return_state=True)
        state = p['initial_state'].clone()
        for t in range(3):
            row = ops.decay_attention_step(p['q'][:, t], p['k'][:, t], p['v'][:, t], p['log_decay'], state)
            assert float((row - whole[:, t]).abs().max()) <= 2.0**-7 * float(whole[:, t].abs().max())     # two roundings
        # both sum the same products in float32 in their own order: a few of 2^-24 of the largest terms
        assert torch.allclose(state, last, rtol=1e-5, atol=1e-5 * float(last.abs().max()))
    p = to_gpu(problem(2, 30, 2, 16, 8, 'f32', seed=16))
    q = p['q'].requires_grad_()
    out = ops.decay_attention(q, p['k'], p['v'], p['log_decay'])
    one = torch.autograd.grad(out, q, p['grad_out'], retain_graph=True)[0]
    assert torch.equal(one, torch.autograd.grad(out, q, p['grad_out'])[0])


@gpu
def test_threads_with_streams_of_their_own():
    """eight threads, each with its own stream and sizes, forward and backward at once: every one gets what it gets alone"""
    import threading

    def work(n, results):
        p = to_gpu(problem(1 + n, 100 + 50 * n, 2, 16 * (n % 3 + 1), 32, ('f32', 'bf16', 'f16')[n % 3], seed=20 + n))
        x, teacher, weight = distill_problem(20 + n, 300 + 400 * n, 9, 'f32', 2.0, seed=20 + n)
        x, teacher, weight = x.cuda().requires_grad_(), teacher.to('cuda'), weight.cuda()
        q = p['q'].requires_grad_()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(5):
                out = ops.decay_attention(q, p['k'], p['v'], p['log_decay'], p.get('lengths'))
                grad = torch.autograd.grad(out, q, p['grad_out'])[0]
                loss = ops.distillation_loss(x, teacher, weight)
                g = torch.autograd.grad(loss, x)[0]
                top = ops.top_logits(x.detach(), 9)
            stream.synchronize()
            results[n] = [y.detach().cpu() for y in (out, grad, loss, g, top.values, top.indices, top.rest)]
    alone, together = {}, {}
    for n in range(8):
        work(n, alone)
    threads = [threading.Thread(target=work, args=(n, together)) for n in range(8)]
    [t.start() for t in threads], [t.join() for t in threads]
    for n in range(8):
        for y, z in zip(together[n], alone[n]):
            assert torch.equal(y, z), n


@gpu
@pytest.mark.parametrize('rows,classes,k', [(500, 5000, 64), (300, 900, 20), (100, 60001, 128)])
def test_top_logits_gives_the_same_bits_again(rows, classes, k):
    """nothing depends on the order in which threads note what they find"""
    x = torch.randn(rows, classes, generator=torch.Generator().manual_seed(3)).cuda()
    first = ops.top_logits(x, k, 0.7)
    for _ in range(20):
        again = ops.top_logits(x, k, 0.7)
        for name in ('values', 'indices', 'rest'):
            assert torch.equal(getattr(first, name), getattr(again, name)), name


@gpu
@pytest.mark.parametrize('dtype', sorted(TYPES))
def test_a_training_pass_gives_the_same_bits_again(dtype):
    """cut into segments, with states, other passes between: and gradients of k and v that are the 64-bit ones rounded once, also
    where the state is returned (all but those next to the middle between two numbers)"""
    shape = (2, 1000, 2, 64, 64)
    p, other = problem(*shape, dtype, True, True, seed=51), to_gpu(problem(*shape, dtype, True, True, seed=52))
    d, bits = to_gpu(p), []
    for turn in range(4):
        for q in (d, other):
            leaves = [q[x].detach().requires_grad_() for x in LEAVES]
            out, state = ops.decay_attention(*leaves[:4], q['lengths'], leaves[4], True)
            grads = torch.autograd.grad([out, state], leaves, [q['grad_out'], q['grad_state']])
            if q is d:
                bits.append([x.detach().clone() for x in (out, state, *grads)])
    assert all(torch.equal(x, y) for b in bits[1:] for x, y in zip(b, bits[0]))
    if dtype != 'f32':
        want = gradients(p)
        for x, got in (('k', bits[0][3]), ('v', bits[0][4])):
            once = want[x].to(TYPES[dtype])
            # sums of float32 and operands of 16 bits move a value by some 2^-16 of its terms: across the middle in 2^-16 / 2^-9 of
            # the cases in bfloat16 (2^-12 in float16), a few times more often where terms cancel
            assert float((got.cpu() != once).double().mean()) < 8 * 2.0 ** -16 / (torch.finfo(TYPES[dtype]).eps / 2), x


@gpu
@pytest.mark.parametrize('classes', [40, 5003, 20001])
@pytest.mark.parametrize('wide', [False, True])
def test_indices_that_changed_behind_the_forward_pass_stay_in_their_rows(classes, wide):
    """the C entries: the backward pass bounds the indices it is given itself; a place that is gone counts among the unlisted"""
    x, teacher, weight = distill_problem(9, classes, 3, 'f32', 2.0, seed=50)
    x, teacher = x.cuda(), teacher.to('cuda')
    indices = teacher.indices.long() if wide else teacher.indices.clone()
    guard, lib = classes * 4, N.load_library()
    held = torch.full((2 * guard + 9 * classes,), 7.0, device='cuda')
    stats, row_loss, one = torch.empty(9, 4 + 3, device='cuda'), torch.empty(9, device='cuda'), torch.ones(9, device='cuda')
    d = N.PxgDistill()
    d.struct_bytes, d.rows, d.classes, d.row_stride, d.k, d.temperature = C.sizeof(d), 9, classes, classes, 3, 2.0
    d.logits, d.values, d.indices, d.rest = (t.data_ptr() for t in (x, teacher.values, indices, teacher.rest))
    d.indices_are_64, d.grad_per_row, d.row_loss, d.stats = int(wide), 1, row_loss.data_ptr(), stats.data_ptr()
    d.grad_loss, d.grad_logits = one.data_ptr(), held.data_ptr() + 4 * guard
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.pxg_distill_forward(C.byref(d), stream) == 0 and lib.pxg_distill_backward(C.byref(d), stream) == 0
    grad = held[guard:-guard].view(9, classes).clone()
    want = ops.distillation_loss_and_gradient(x, teacher, None, 'none')
    assert torch.equal(row_loss, want[0]) and torch.equal(grad, want[1])
    gone = [(0, 0, classes), (3, 1, -1), (5, 2, -2), (8, 0, classes * 2), (8, 1, -classes)] + ([(6, 0, 1 << 40)] if wide else [])
    for row, place, index in gone:
        indices[row, place] = index
    held.fill_(7.0)
    assert lib.pxg_distill_backward(C.byref(d), stream) == 0
    got = held[guard:-guard].view(9, classes)
    assert (held[:guard] == 7.0).all() and (held[-guard:] == 7.0).all()
    same = torch.ones_like(got, dtype=torch.bool)
    for row, place, index in gone:
        same[row, int(teacher.indices[row, place])] = False
    assert torch.equal(got[same], grad[same]) and torch.isfinite(got).all()


@gpu
def test_more_rows_than_one_axis_of_a_grid_holds():
    rows = (1 << 26) + 5                                           # four to a workgroup of 256: 2^32 threads and more
    x = torch.randn(rows, 2, device='cuda', generator=torch.Generator('cuda').manual_seed(4))
    t = ops.top_logits(x, 1)
    want, at = x.max(dim=1)
    assert torch.equal(t.values[:, 0], want) and torch.equal(t.indices[:, 0], at.int())
    assert torch.allclose(t.rest, x.min(dim=1).values, rtol=1e-6, atol=1e-6)
    student = torch.stack([x[:, 1], x[:, 0]], dim=1)
    loss, grad = ops.distillation_loss_and_gradient(student, t, reduction='none')
    for part in (slice(0, 1000), slice((1 << 26) - 500, rows)):    # softmaxes of two, in 64 bits
        p, q = x[part].double().log_softmax(1), student[part].double().log_softmax(1)
        assert torch.allclose(loss[part].double(), (p.exp() * (p - q)).sum(1), rtol=1e-5, atol=1e-6)
        assert torch.allclose(grad[part].double(), q.exp() - p.exp(), rtol=1e-5, atol=1e-6)


@gpu
def test_offsets_beyond_32_bits():
    """rows behind the 2^31st element are computed as they are alone (the same kernels on the same numbers: the same bits, or, where
    an earlier memory of exp(-2000) is left out or the time axis is cut elsewhere, two roundings of the result)"""
    g = torch.Generator('cuda').manual_seed(5)
    normal = lambda *shape, dtype=torch.bfloat16: torch.randn(*shape, device='cuda', dtype=dtype, generator=g)          # noqa: E731
    steps, tail = (1 << 20) + 77, 2048                             # 16 heads of 128: 2^31 elements and more
    q, k, v, go = (normal(1, steps, 16, 128) for _ in range(4))
    log_decay = torch.full((16,), -1.0, device='cuda')

    def last(t):
        return t[:, -tail:].contiguous()
    out = ops.decay_attention(q, k, v, log_decay)
    near = lambda x, y: bool(((x.float() - y.float()).abs() <= 2.0**-7 * y.float().abs() + 2.0**-9 * y.float().abs().max()).all())  # noqa: E731
    alone = ops.decay_attention(last(q), last(k), last(v), log_decay)
    assert near(out[:, -1000:], alone[:, -1000:])
    del out
    grads = ops.decay_attention_backward(go, q, k, v, log_decay)[:3]
    alone = ops.decay_attention_backward(last(go), last(q), last(k), last(v), log_decay)[:3]
    for x, y in zip(grads, alone):
        assert near(x[:, -1000:], y[:, -1000:])
    del q, k, v, go, grads
    # sequences that lie so far apart, and steps of a stride that no 32-bit offset inside a chunk holds
    store = torch.empty((1 << 31) + (1 << 20), device='cuda', dtype=torch.bfloat16)
    p = to_gpu(problem(2, 70, 2, 64, 64, 'bf16', True, seed=6))
    want = ops.decay_attention(p['q'], p['k'], p['v'], p['log_decay'], p['lengths'])
    far = store.as_strided((2, 70, 2, 64), (1 << 31, 128, 64, 1))
    far.copy_(p['k'])
    assert torch.equal(ops.decay_attention(p['q'], far, p['v'], p['log_decay'], p['lengths']), want)
    apart = store.as_strided((2, 70, 2, 64), (128, 1 << 24, 64, 1))
    apart.copy_(p['v'])
    assert torch.equal(ops.decay_attention(p['q'], p['k'], apart, p['log_decay'], p['lengths']), want)
    del store, far, apart
    # many states, many logits
    pairs = 131072 + 3
    state, first = torch.empty(pairs, 1, 128, 128, device='cuda').normal_(generator=g), normal(3, 1, 128)
    one = state[-3:].clone()
    x = first[:1].expand(pairs, 1, 128).clone()
    x[-3:] = first
    got = ops.decay_attention_step(x, x, x, log_decay[:1], state)
    assert torch.equal(got[-3:], ops.decay_attention_step(first, first, first, log_decay[:1], one)) and torch.equal(state[-3:], one)
    del state, x, got
    rows = (1 << 16) + 300
    logits = normal(rows, 32768)                                   # (2 100 of them go the way of all)
    t = ops.top_logits(logits, 20)
    end = ops.top_logits(logits[-2100:].contiguous(), 20)
    assert torch.equal(t.values[-2100:], end.values) and torch.equal(t.indices[-2100:], end.indices) and torch.equal(t.rest[-2100:], end.rest)
    loss, grad = ops.distillation_loss_and_gradient(logits, ops.TopLogits(t.values * 2, t.indices, t.rest), None, 'none')
    end = ops.distillation_loss_and_gradient(logits[-2100:].contiguous(), ops.TopLogits(end.values * 2, end.indices, end.rest), None, 'none')
    assert torch.equal(loss[-2100:], end[0]) and torch.equal(grad[-2100:], end[1])


# ---- refusals (on the CPU: nothing is launched) -------------------------------------------------------------------------
@pytest.fixture
def dry(monkeypatch):
    """the checks of arguments alone: CPU tensors pass as GPU tensors, a launch fails the test"""
    monkeypatch.setattr(ops, '_on_gpu', lambda name, t, device=None: None)

    def launched(*a):
        raise AssertionError('launched')
    monkeypatch.setattr(ops, '_ext', launched)


def test_cpu_tensors_are_refused():
    p = problem(1, 4, 1, 8, 8, 'f32')
    with pytest.raises(ValueError, match='on a GPU only'):
        ops.decay_attention(*[p[x] for x in ARGS[:4]])
    with pytest.raises(ValueError, match='on a GPU only'):
        ops.top_logits(torch.zeros(2, 3), 1)
    with pytest.raises(ValueError, match='on a GPU only'):
        ops.distillation_loss(torch.zeros(2, 3), ops.TopLogits(torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int32)))
    with pytest.raises(TypeError, match='must be a tensor'):
        ops.top_logits([[1.0]], 1)


def test_decay_refusals(dry):
    p = problem(2, 4, 3, 8, 6, 'f32', state=True)
    args = {x: p[x] for x in ARGS}
    for change, error, text in [
            ({'k': p['k'].bfloat16()}, TypeError, 'k is'), ({'q': p['q'].double()}, TypeError, 'float32, bfloat16 or float16'),
            ({'q': p['q'][0]}, ValueError, 'q, k and v'), ({'k': p['k'][..., :7]}, ValueError, 'q, k and v'),
            ({'v': p['v'][:, :3]}, ValueError, 'q, k and v'), ({'v': p['v'][:, :, :2]}, ValueError, 'q, k and v'),
            ({'v': torch.zeros(2, 4, 3, 129)}, ValueError, 'widths'), ({'v': torch.zeros(2, 4, 3, 0)}, ValueError, 'widths'),
            ({'log_decay': p['log_decay'][:2]}, ValueError, 'log_decay'), ({'log_decay': p['log_decay'].double()}, TypeError, 'log_decay'),
            ({'lengths': torch.ones(2)}, TypeError, 'lengths'), ({'lengths': torch.ones(3, dtype=torch.int32)}, ValueError, 'lengths'),
            ({'initial_state': p['initial_state'].half()}, TypeError, 'initial_state'),
            ({'initial_state': p['initial_state'].transpose(2, 3)}, ValueError, 'initial_state')]:
        with pytest.raises(error, match=text):
            ops.decay_attention(**{**args, **change})
    with pytest.raises(ValueError, match='grad_out'):
        ops.decay_attention_backward(p['grad_out'][:, :3], **args)
    with pytest.raises(ValueError, match='grad_state'):
        ops.decay_attention_backward(p['grad_out'], **args, grad_state=p['grad_state'][:1])
    one = {x: p[x][:, 0] for x in ('q', 'k', 'v')}
    step = {**one, 'log_decay': p['log_decay'], 'state': p['initial_state']}
    for change, error, text in [({'q': p['q']}, ValueError, 'q, k and v'), ({'state': p['initial_state'][:1]}, ValueError, 'state'),
                                ({'state': p['initial_state'].transpose(2, 3).contiguous().transpose(2, 3)}, ValueError, 'contiguous'),
                                ({'active': torch.ones(2)}, ValueError, 'active'), ({'active': torch.ones(3).bool()}, ValueError, 'active'),
                                ({'q': one['q'].clone().requires_grad_()}, RuntimeError, 'no gradients')]:
        with pytest.raises(error, match=text):
            ops.decay_attention_step(**{**step, **change})


def test_distillation_refusals(dry):
    x = torch.zeros(4, 9)
    good = ops.TopLogits(torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4), 2.0)
    for logits, k, temperature, error, text in [
            (x.double(), 2, 1.0, TypeError, 'float32'), (x[0], 2, 1.0, ValueError, 'rows, classes'), (x, 0, 1.0, ValueError, 'k is'),
            (x, 10, 1.0, ValueError, 'k is'), (torch.zeros(2, 200), 129, 1.0, ValueError, 'k is'), (x, 2, 0.0, ValueError, 'temperature'),
            (x, 2, float('nan'), ValueError, 'temperature'), (x, 2, float('inf'), ValueError, 'temperature'),
            (torch.zeros(4, 0), 1, 1.0, ValueError, 'rows, classes')]:
        with pytest.raises(error, match=text):
            ops.top_logits(logits, k, temperature)
    t = good
    for logits, teacher, options, error, text in [
            (x.double(), t, {}, TypeError, 'float32'), (x, (t.values, t.indices), {}, TypeError, 'TopLogits'),
            (x[:3], t, {}, ValueError, 'teacher.values'), (x, ops.TopLogits(t.values, t.indices.float(), t.rest), {}, TypeError, 'indices'),
            (x, ops.TopLogits(t.values, t.indices[:, :2], t.rest), {}, ValueError, 'teacher.values'),
            (x, ops.TopLogits(t.values, t.indices, t.rest.double()), {}, TypeError, 'rest'),
            (x, ops.TopLogits(t.values, t.indices, t.rest[:2]), {}, ValueError, 'rest'),
            (x, ops.TopLogits(t.values, t.indices, t.rest, -1.0), {}, ValueError, 'temperature'),
            (x, ops.TopLogits(torch.zeros(4, 129), torch.zeros(4, 129).int(), t.rest), {}, ValueError, 'up to 128'),
            (x, t, {'weight': torch.zeros(3)}, ValueError, 'weight'), (x, t, {'weight': torch.zeros(4).half()}, TypeError, 'weight'),
            (x, t, {'weight': torch.zeros(4, requires_grad=True)}, ValueError, 'gradient'),
            (x, t, {'reduction': 'avg'}, ValueError, 'reduction')]:
        with pytest.raises(error, match=text):
            ops.distillation_loss(logits, teacher, **options)
    with pytest.raises(ValueError, match='grad_loss'):
        ops.distillation_loss_and_gradient(x, t, grad_loss=torch.zeros(4))


def test_top_logits_rows():
    t = ops.TopLogits(torch.arange(8.0).view(4, 2), torch.arange(8).view(4, 2), torch.arange(4.0), 2.0)
    assert len(t) == 4 and t[torch.tensor([2, 0])].rest.tolist() == [2.0, 0.0] and t[1].values.tolist() == [[2.0, 3.0]]
    assert t[-1].indices.tolist() == [[6, 7]] and t.to('cpu').temperature == 2.0 and t[1:3].temperature == 2.0
    both = ops.TopLogits.cat([t[:1], t[1:]])
    assert both.values.equal(t.values) and both.rest.equal(t.rest)
    with pytest.raises(ValueError, match='temperatures'):
        ops.TopLogits.cat([t, ops.TopLogits(t.values, t.indices, t.rest, 1.0)])
    assert ops.TopLogits(t.values, t.indices)[0].rest is None


@pytest.fixture
def idle(monkeypatch):
    """the extension over entry points that do nothing but fail: CPU tensors pass as GPU tensors, nothing is ever launched"""
    monkeypatch.setattr(ops, '_on_gpu', lambda name, t, device=None: None)
    ext, lib = ops._ext(), N.load_library()
    fails = C.CFUNCTYPE(C.c_int64)(lambda: -1)
    ext.use_library([C.cast(fails, C.c_void_p).value] * len(ops._ENTRY_POINTS))
    yield
    ext.use_library([C.cast(getattr(lib, name), C.c_void_p).value for name in ops._ENTRY_POINTS])


def every_call(p, change=lambda name, t: t):
    """(name, call) of every public call, with `change` made to one tensor at a time"""
    x, teacher, weight = distill_problem(3, 9, 2, 'f32', 2.0, seed=43)
    step = {n: p[n][:, 0] for n in 'qkv'}
    for n in ARGS + ('grad_out', 'grad_state'):
        if p[n].is_floating_point():
            if n in ARGS:
                yield 'decay_attention', lambda n=n: ops.decay_attention(**{m: change(m, p[m]) if m == n else p[m] for m in ARGS})
                if n in step or n == 'log_decay':
                    yield 'decay_attention_step', lambda n=n: ops.decay_attention_step(**{**step, 'log_decay': p['log_decay'], n: change(
                        n, step.get(n, p['log_decay']))}, state=p['initial_state'])
            yield 'decay_attention_backward', lambda n=n: ops.decay_attention_backward(**{m: change(m, p[m]) if m == n else p[m] for m in ARGS + (
                'grad_out', 'grad_state')})
    yield 'decay_attention_step', lambda: ops.decay_attention_step(**step, log_decay=p['log_decay'], state=change('state', p['initial_state']))
    dev = p['q'].device
    call = {'logits': x.to(dev), 'values': teacher.values.to(dev), 'rest': teacher.rest.to(dev), 'weight': weight.to(dev)}
    for n in call:
        for name in ('distillation_loss', 'distillation_loss_and_gradient'):
            def one(name=name, n=n):
                c = {**call, n: change(n, call[n])}
                return getattr(ops, name)(c['logits'], ops.TopLogits(c['values'], teacher.indices.to(dev), c['rest'], 2.0), c['weight'])
            yield name, one


def tangents_are_refused(p):
    fw, seen = torch.autograd.forward_ad, set()
    with fw.dual_level():
        for name, call in every_call(p, lambda n, t: fw.make_dual(t, torch.ones_like(t))):
            with pytest.raises(NotImplementedError, match=name + ' has no forward-mode derivative'):
                call()
            seen.add(name)
    assert len(seen) == 5


def test_tangents_are_refused(idle):
    tangents_are_refused(problem(2, 4, 1, 8, 8, 'f32', True, True, seed=42))


@gpu
def test_tangents_are_refused_on_the_gpu():
    p = to_gpu(problem(2, 4, 1, 8, 8, 'f32', True, True, seed=42))
    tangents_are_refused(p)
    with torch.autograd.forward_ad.dual_level():                    # numbers without a tangent are no matter of it
        assert torch.isfinite(ops.decay_attention(**{n: p[n] for n in ARGS})).all()


def test_temperatures_below_the_least_normal_number_are_refused(dry):
    lib = N.load_library()
    d = N.PxgDistill()
    d.struct_bytes, d.rows, d.classes, d.k = C.sizeof(d), 0, 8, 0
    for tau in (1e-39, 1e-50, 1.1e-38, -1.0, 3.1e38):
        with pytest.raises(ValueError, match='temperature'):
            ops.top_logits(torch.zeros(2, 3), 1, tau)
        with pytest.raises(ValueError, match='temperature'):
            ops.distillation_loss(torch.zeros(2, 3), ops.TopLogits(torch.zeros(2, 1), torch.zeros(2, 1).int(), None, tau))
        d.temperature = tau
        assert lib.pxg_distill_forward(C.byref(d), None) == -1 and lib.pxg_top_logits(0, 0, 8, None, 8, 2, tau, None, None, None, None) == -1
    for tau in (1.2e-38, 1.0, 3e38):
        d.temperature = tau
        assert lib.pxg_distill_forward(C.byref(d), None) == 0 and lib.pxg_top_logits(0, 0, 8, None, 8, 2, tau, None, None, None, None) == 0


@gpu
def test_extreme_temperatures():
    for classes in (9, 300):
        x = torch.zeros(2, classes)
        x[:, 0], x[1, 1:] = 1.0, torch.linspace(-1.0, 0.0, classes - 1)
        for tau in (1.2e-38, 3e38):
            t = ops.top_logits(x.cuda(), 1, tau)
            # equal ones: their number; else the largest counts alone, or all do
            want = [math.log(classes - 1), 0.0 if tau < 1 else math.log(classes - 1)]
            assert t.indices[:, 0].tolist() == [0, 0] and np.allclose(t.rest.cpu().numpy(), want, atol=1e-6)
            # the listed class far ahead of all others, or as good as each of them
            loss, grad = ops.distillation_loss_and_gradient(x.cuda(), t, reduction='none')
            assert torch.isfinite(grad).all() and float(loss.abs().max()) <= (1e-30 if tau < 1 else math.inf)


def refused_state(p):
    with torch.inference_mode():
        state = p['initial_state'].clone()
    with pytest.raises(RuntimeError, match='[Ii]nference'):
        ops.decay_attention_step(*[p[n][:, 0] for n in 'qkv'], p['log_decay'], state)
    return state


def test_a_state_of_inference_mode_is_refused_outside_it(idle):
    refused_state(problem(2, 4, 1, 8, 8, 'f32', True, True, seed=45))      # (had it been launched, another error)


@gpu
def test_a_refused_state_is_left_as_it_was():
    p = to_gpu(problem(2, 4, 1, 8, 8, 'f32', True, True, seed=45))
    assert torch.equal(refused_state(p), p['initial_state'])


def recordings_are_refused(p):
    from torch.fx.experimental.proxy_tensor import make_fx
    calls, seen = list(every_call(p)), set()
    calls.append(('top_logits', lambda: ops.top_logits(p['q'][:, 0, 0], 3).values))
    for name, call in calls:
        if name in seen:
            continue
        seen.add(name)
        with pytest.raises(NotImplementedError, match=name + ' cannot be traced'):
            torch.jit.trace(lambda x: (call(), x)[1], p['q'], check_trace=False)
        with pytest.raises(NotImplementedError, match=name + ' cannot be traced'):
            make_fx(lambda x: (call(), x)[1])(p['q'])
    assert len(seen) == 6


@pytest.mark.filterwarnings('ignore::torch.jit.TracerWarning')
def test_recordings_are_refused(idle):
    recordings_are_refused(problem(2, 4, 1, 8, 8, 'f32', True, True, seed=44))


@gpu
@pytest.mark.filterwarnings('ignore::torch.jit.TracerWarning')
def test_recordings_are_refused_on_the_gpu():
    p = to_gpu(problem(2, 4, 1, 8, 8, 'f32', True, True, seed=44))
    recordings_are_refused(p)
    assert torch.isfinite(ops.decay_attention(**{n: p[n] for n in ARGS})).all()
    # what breaks a graph at such a call instead of recording through it goes on as it did
    want = ops.decay_attention(**{n: p[n] for n in ARGS}) * 2
    got = torch.compile(lambda q: ops.decay_attention(**{**{n: p[n] for n in ARGS}, 'q': q}) * 2, backend='eager')(p['q'])
    assert torch.equal(got, want)


def test_answers_one_row_after_the_other():
    t = ops.TopLogits(torch.arange(8.0).view(4, 2), torch.arange(8).view(4, 2), torch.arange(4.0), 2.0)
    rows = []
    for row in t:
        rows.append(row)
        assert len(rows) <= 4
    assert ops.TopLogits.cat(rows).values.equal(t.values) and ops.TopLogits.cat(rows).rest.equal(t.rest)
    assert t[np.int64(2)].values.equal(t.values[2:3]) and t[np.int64(-1)].rest.equal(t.rest[3:])
    for at in (4, -5, np.int64(4)):
        with pytest.raises(IndexError, match='of 4'):
            t[at]


def mixed_parts():
    x, t, weight = distill_problem(6, 40, 3, 'f32', 2.0, seed=41)
    return x, weight, [t[:2], ops.TopLogits(t.values[2:5], t.indices[2:5], None, 2.0), t[5:]], t


def test_answers_with_and_without_a_rest_are_joined():
    x, weight, parts, t = mixed_parts()
    for order in ([0, 1, 2], [1, 0, 2], [1, 2]):
        both = ops.TopLogits.cat([parts[i] for i in order])
        want = torch.cat([torch.full((3,), -math.inf) if i == 1 else parts[i].rest for i in order])
        assert both.rest.equal(want) and both.rest.dtype == torch.float32 and both.values.equal(torch.cat([parts[i].values for i in order]))
    assert ops.TopLogits.cat([parts[1], parts[1]]).rest is None
    assert ops.TopLogits.cat([t[:0], parts[1]]).rest.equal(torch.full((3,), -math.inf))


@gpu
def test_joined_answers_have_the_losses_of_their_parts():
    x, weight, parts, _ = mixed_parts()
    x, weight, parts = x.cuda(), weight.cuda(), [p.to('cuda') for p in parts]
    loss, grad = ops.distillation_loss_and_gradient(x, ops.TopLogits.cat(parts), weight, 'none')
    rows = torch.arange(6).split([2, 3, 1])
    alone = [ops.distillation_loss_and_gradient(x[r], p, weight[r], 'none') for r, p in zip(rows, parts)]
    assert torch.equal(loss, torch.cat([a for a, _ in alone])) and torch.equal(grad, torch.cat([b for _, b in alone]))


def test_c_entries_refuse_what_they_can_see():
    """bad shapes, types and missing pointers come back as PXG_E_INVALID before anything touches a GPU"""
    lib = N.load_library()
    invalid = -1
    s = N.PxgDecay()
    assert lib.pxg_decay_forward(C.byref(s), None) == invalid                     # struct_bytes
    s.struct_bytes, s.batch, s.steps, s.heads, s.dk, s.dv = C.sizeof(s), 1, 1, 1, 8, 8
    for fn in (lib.pxg_decay_forward, lib.pxg_decay_backward, lib.pxg_decay_step):
        assert fn(C.byref(s), None) == invalid and fn(None, None) == invalid      # no pointers
    for field, value in (('dtype', 3), ('dk', 129), ('dk', 0), ('dv', -1), ('heads', 0), ('batch', -1), ('steps', -1),
                         ('batch', 1 << 40), ('steps', 1 << 40)):
        t = N.PxgDecay.from_buffer_copy(s)
        setattr(t, field, value)
        assert lib.pxg_decay_workspace_bytes(C.byref(t), 1) == invalid, field
    t = N.PxgDecay.from_buffer_copy(s)
    t.batch, t.log_decay = 0, 4096
    assert lib.pxg_decay_forward(C.byref(t), None) == 0                           # nothing to do
    d = N.PxgDistill()
    assert lib.pxg_distill_forward(C.byref(d), None) == invalid
    d.struct_bytes, d.rows, d.classes, d.temperature, d.k = C.sizeof(d), 1, 8, 1.0, 2
    assert lib.pxg_distill_forward(C.byref(d), None) == invalid and lib.pxg_distill_backward(C.byref(d), None) == invalid
    d.rows = 0
    assert lib.pxg_distill_forward(C.byref(d), None) == 0 and lib.pxg_distill_backward(C.byref(d), None) == 0
    for field, value in (('k', 129), ('k', -1), ('classes', 0), ('temperature', 0.0), ('temperature', float('nan')), ('dtype', -1),
                         ('value_dtype', 7)):
        e = N.PxgDistill.from_buffer_copy(d)
        setattr(e, field, value)
        assert lib.pxg_distill_forward(C.byref(e), None) == invalid, field
    top = lambda dt=0, rows=1, classes=8, k=2, tau=1.0: lib.pxg_top_logits(dt, rows, classes, None, 8, k, tau, None, None, None, None)  # noqa: E731
    assert top() == top(rows=-1) == top(k=0) == top(k=9) == top(tau=0.0) == top(dt=5) == invalid and top(rows=0) == 0


def test_structs_match_the_header():
    import os
    import subprocess
    import tempfile
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = '#include <stdio.h>\n#include "pxg.h"\nint main(){printf("%zu %zu %zu", sizeof(pxg_sequence), sizeof(pxg_decay), sizeof(pxg_distill));return 0;}'
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, 'sz.c'), 'w').write(src)
        exe = os.path.join(d, 'sz')
        subprocess.check_call(['gcc', '-I' + os.path.join(root, 'include'), os.path.join(d, 'sz.c'), '-o', exe])
        sizes = [int(v) for v in subprocess.check_output([exe]).split()]
    assert sizes == [C.sizeof(N.PxgSequence), C.sizeof(N.PxgDecay), C.sizeof(N.PxgDistill)]


def test_more_pairs_than_a_grid_holds(dry):
    """refused by the checks and by the C entries (views of one element: nothing of that size exists)"""
    q = torch.zeros(1, 1, 1, 1).expand(1 << 22, 1, 2, 1)
    with pytest.raises(ValueError, match='at most'):
        ops.decay_attention(q, q, q, torch.zeros(2))
    s = N.PxgDecay()
    s.struct_bytes, s.batch, s.steps, s.heads, s.dk, s.dv = C.sizeof(s), 1 << 22, 1, 2, 1, 1
    lib = N.load_library()
    assert lib.pxg_decay_workspace_bytes(C.byref(s), 0) == -1
    s.batch -= 1
    assert lib.pxg_decay_workspace_bytes(C.byref(s), 0) == 0
    s.batch, s.heads = 0, 1 << 24
    assert lib.pxg_decay_workspace_bytes(C.byref(s), 0) == -1


def test_answers_are_moved_never_cast():
    t = ops.TopLogits(torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3), 2.0)
    for to in (torch.float16, 'cpu', torch.device('cpu'), torch.empty(1, dtype=torch.float64)):
        moved = t.to(to)
        assert moved.values.dtype == torch.float32 and moved.indices.dtype == torch.int32 and moved.temperature == 2.0
    meta = ops.TopLogits(torch.zeros(3, 2, device='meta'), torch.zeros(3, 2, dtype=torch.int32, device='meta')).to(torch.float16)
    assert meta.values.device.type == 'meta'
