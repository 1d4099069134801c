"""The sequence and distillation operators of poreplex_amd.torch_ops as measurable cases.

Four operators, in their plain form (elementary torch operations in 32 bits) and through the framework's entry points:

  attention   decay_attention          o_t = q_t S_t,  S_t = exp(log_decay) S_{t-1} + k_t v_t^T, whole sequences, per head;
                                       with "train": its gradients for q, k, v, log_decay and the initial state
  step        decay_attention_step     one token of the same recurrence, the state updated in place
  top         top_logits               a teacher's k largest logits per row, their classes, and the log-sum-exp of the rest
  distill     distillation_loss        tau^2 KL(teacher || student) over the listed classes and one bucket for the rest,
                                       with its gradient for the student's logits

Widths and lengths are this package's own where it has them (300-step barcode windows, 2 000-step read heads, 256-sample training batches,
10 000-read batches, 5 classes, 64 units); the rest are generic.
"""
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
CHUNK = 64


def listed():
    return [
        # a training batch's windows through one recurrent layer, at evaluation
        attention('windows-f32', 256, 300, 4, 16, 16, 'f32'),
        # read heads of different lengths in one padded batch; the state is kept for the samples that follow
        attention('heads-ragged-bf16', 128, 2000, 8, 64, 64, 'bf16', ragged=True, state=True),
        # one very long signal that goes on from an earlier state: few rows, a long axis
        attention('long-f16', 1, 100003, 8, 128, 128, 'f16', state=True),
        # one training step of the layer on a batch of windows
        attention('windows-train-f32', 256, 300, 4, 16, 16, 'f32', train=True),
        # training on read heads with carried states (truncated back-propagation)
        attention('heads-train-bf16', 16, 2000, 8, 64, 64, 'bf16', ragged=True, state=True, train=True),
        # a single stream's next token: latency
        step('step-one-bf16', 1, 4, 64, 64, 'bf16', active=False),
        # every channel of a large run, some of them idle
        step('step-channels-bf16', 2048, 8, 64, 64, 'bf16', active=True),
        # a teacher's answers for a 10 000-read batch of the barcode classifier
        top('top-barcodes-f32', 10000, 5, 3, 'f32', 2.0),
        # a teacher with many classes, an odd number of them
        top('top-wide-bf16', 2047, 50001, 64, 'bf16', 1.0),
        # the loss of one training batch of the barcode classifier
        distill('distill-barcodes-f32', 256, 5, 3, 'f32', 2.0),
        # many classes, half precision
        distill('distill-wide-bf16', 4096, 32768, 32, 'bf16', 1.0),
        # the widest rows, odd, in full precision
        distill('distill-widest-f32', 1023, 131071, 100, 'f32', 4.0),
    ]


def attention(name, batch, steps, heads, dk, dv, dtype, ragged=False, state=False, train=False):
    return named(name, op='attention', batch=batch, steps=steps, heads=heads, dk=dk, dv=dv, dtype=dtype, ragged=ragged, state=state,
                 train=train)


def step(name, batch, heads, dk, dv, dtype, active):
    return named(name, op='step', batch=batch, heads=heads, dk=dk, dv=dv, dtype=dtype, active=active)


def top(name, rows, classes, k, dtype, temperature):
    return named(name, op='top', rows=rows, classes=classes, k=k, dtype=dtype, temperature=temperature)


def distill(name, rows, classes, k, dtype, temperature):
    return named(name, op='distill', rows=rows, classes=classes, k=k, dtype=dtype, temperature=temperature)


def named(name, **case):
    if name is not None:
        case['name'] = name
    return case


def spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(['attention', 'attention', 'step', 'top', 'distill'])
    dtype = rng.choice(sorted(DTYPES))
    if op in ('attention', 'step'):
        dk, dv = rng.choice([16, 24, 32, 48, 64, 80, 128]), rng.choice([16, 32, 40, 48, 64, 128])
        heads = rng.randint(1, 8)
        if op == 'step':
            return step(None, spread(rng, 1, 2048 * 8 * 64 * 64 // (heads * dk * dv)), heads, dk, dv, dtype, rng.random() < 0.5)
        train = rng.random() < 0.5
        steps = spread(rng, 1, 20000 if train else 100000)
        room = (6 << 20 if train else 40 << 20) // (steps * heads * max(dk, dv))     # no more values than the largest listed case
        return attention(None, spread(rng, 1, max(1, min(512, room))), steps, heads, dk, dv, dtype, rng.random() < 0.5,
                         rng.random() < 0.5, train)
    classes = spread(rng, 2, 131071)
    rows = spread(rng, 1, max(1, min(20000, (100 << 20) // classes)))
    k = spread(rng, 1, min(classes, 128))
    return (top if op == 'top' else distill)(None, rows, classes, k, dtype, rng.choice([1.0, 1.5, 2.0, 4.0]))


# ---- what a program has in hand before the call ---------------------------------------------------------------------
def generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, device='cuda', generator=g)


def prepare(case, seed):
    g, dt = generator(seed), DTYPES[case['dtype']]
    if case['op'] in ('attention', 'step'):
        b, h, dk, dv = case['batch'], case['heads'], case['dk'], case['dv']
        # windows of about 8 to 256 tokens over the heads
        spans = 3.0 + 5.0 * (torch.arange(h, device='cuda') + torch.rand(h, device='cuda', generator=g)) / h
        s = {'case': case, 'log_decay': torch.log1p(-torch.exp2(-spans)).float()}
        if case['op'] == 'step':
            s['q'], s['k'] = (normal(g, b, h, dk) * dk ** -0.5).to(dt), normal(g, b, h, dk).to(dt)
            s['v'] = normal(g, b, h, dv).to(dt)
            s['state'] = normal(g, b, h, dk, dv) * 3
            s['active'] = torch.rand(b, device='cuda', generator=g) < 0.9 if case['active'] else None
            return s
        t = case['steps']
        s['q'], s['k'] = (normal(g, b, t, h, dk) * dk ** -0.5).to(dt), normal(g, b, t, h, dk).to(dt)
        s['v'] = normal(g, b, t, h, dv).to(dt)
        s['lengths'] = None
        if case['ragged']:
            s['lengths'] = torch.randint((t + 1) // 2, t + 1, (b,), device='cuda', generator=g).to(torch.int32)
        s['initial_state'] = normal(g, b, h, dk, dv) * 3 if case['state'] else None
        if case['train']:
            s['grad_out'] = normal(g, b, t, h, dv).to(dt)
            s['grad_state'] = normal(g, b, h, dk, dv) if case['state'] else None
            for name in ('q', 'k', 'v', 'log_decay', 'initial_state'):
                if s[name] is not None:
                    s[name].requires_grad_()
        return s
    n, classes, k = case['rows'], case['classes'], case['k']
    logits = normal(g, n, classes) * 3
    if case['op'] == 'top':
        return {'case': case, 'logits': logits.to(dt)}
    student = (logits + normal(g, n, classes)).to(dt)
    values, indices, rest = plain_top(logits.to(dt), k, case['temperature'])
    weight = torch.rand(n, device='cuda', generator=g) * (torch.rand(n, device='cuda', generator=g) < 0.9)
    # half precision trains with a scaled loss, so that small gradients stay above the type's least value
    scale = torch.tensor(1024.0 * n if case['dtype'] == 'f16' else 1.0, device='cuda')
    return {'case': case, 'logits': student.requires_grad_(), 'values': values, 'indices': indices, 'rest': rest, 'weight': weight,
            'grad_loss': scale}


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    case = s['case']
    if case['op'] == 'attention':
        return run_attention(s, case)
    if case['op'] == 'step':
        return run_step(s)
    if case['op'] == 'top':
        return run_top(s, case)
    return run_distill(s, case)


def run_attention(s, case):
    if own:
        from poreplex_amd import torch_ops
        call = torch_ops.decay_attention
    else:
        call = plain_attention
    inputs = [s[x] for x in ('q', 'k', 'v', 'log_decay')]
    options = dict(lengths=s['lengths'], initial_state=s['initial_state'], return_state=case['state'])
    if not case['train']:
        with torch.no_grad():
            got = call(*inputs, **options)
        return dict(zip(('out', 'state'), got if case['state'] else (got,)))
    got = call(*inputs, **options)
    if not case['state']:
        return dict(zip(('out', 'gq', 'gk', 'gv', 'glog_decay'), (got,) + torch.autograd.grad(got, inputs, s['grad_out'])))
    grads = torch.autograd.grad(got, inputs + [s['initial_state']], [s['grad_out'], s['grad_state']])
    return dict(zip(('out', 'state', 'gq', 'gk', 'gv', 'glog_decay', 'ginitial_state'), got + grads))


def run_step(s):
    if own:
        from poreplex_amd import torch_ops
        out = torch_ops.decay_attention_step(s['q'], s['k'], s['v'], s['log_decay'], s['state'], active=s['active'])
    else:
        out = plain_step(s['q'], s['k'], s['v'], s['log_decay'], s['state'], s['active'])
    return {'out': out, 'state': s['state']}


def run_top(s, case):
    if own:
        from poreplex_amd import torch_ops
        t = torch_ops.top_logits(s['logits'], case['k'], temperature=case['temperature'])
        return {'values': t.values, 'indices': t.indices, 'rest': t.rest}
    values, indices, rest = plain_top(s['logits'], case['k'], case['temperature'])
    return {'values': values, 'indices': indices, 'rest': rest}


def run_distill(s, case):
    if own:
        from poreplex_amd import torch_ops
        teacher = torch_ops.TopLogits(s['values'], s['indices'], s['rest'], case['temperature'])
        loss = torch_ops.distillation_loss(s['logits'], teacher, weight=s['weight'])
        return {'loss': loss.detach(), 'grad': torch.autograd.grad(loss, s['logits'], s['grad_loss'])[0]}
    with torch.no_grad():
        loss, grad = plain_distill(s['logits'], s['values'], s['indices'], s['rest'], case['temperature'], s['weight'], s['grad_loss'])
    return {'loss': loss, 'grad': grad}


# ---- plain forms ----------------------------------------------------------------------------------------------------
def plain_attention(q, k, v, log_decay, lengths=None, initial_state=None, return_state=False):
    """Chunks of 64 tokens: a masked product inside each, the states at their borders as one decayed triangular product."""
    b, t, h, dk = q.shape
    dv, n = v.shape[-1], -(-t // CHUNK)
    f = torch.float32
    pos = torch.arange(t, device=q.device)
    length = torch.full((b,), t, device=q.device) if lengths is None else lengths.long()
    live = (pos < length[:, None])[:, :, None, None]

    def chunks(x):
        x = torch.where(live, x.to(f), torch.zeros((), device=x.device))
        pad = torch.zeros(b, n * CHUNK - t, h, x.shape[-1], device=x.device)
        return torch.cat([x, pad], 1).view(b, n, CHUNK, h, -1).permute(0, 3, 1, 2, 4).contiguous()       # b h n c d
    qc, kc, vc = chunks(q), chunks(k), chunks(v)
    i = torch.arange(CHUNK, device=q.device)
    ahead = i[:, None] - i[None, :]
    decay = torch.exp(ahead.clamp(min=0) * log_decay[:, None, None]) * (ahead >= 0)                     # h c c
    out = (qc @ kc.transpose(-1, -2).contiguous() * decay[:, None]) @ vc
    tail = torch.exp((CHUNK - 1 - i) * log_decay[:, None])                                               # h c
    local = (kc * tail[:, None, :, None]).transpose(-1, -2).contiguous() @ vc                            # b h n dk dv
    m = torch.arange(n, device=q.device)
    gap = m[:, None] - 1 - m[None, :]
    carry = torch.exp(CHUNK * gap.clamp(min=0) * log_decay[:, None, None]) * (gap >= 0)                 # h n n
    before = (carry @ local.reshape(b, h, n, dk * dv)).view(b, h, n, dk, dv)
    if initial_state is not None:
        before = before + torch.exp(CHUNK * m * log_decay[:, None])[:, :, None, None] * initial_state[:, :, None]
    head = torch.exp((i + 1) * log_decay[:, None])
    out = out + (qc * head[:, None, :, None]) @ before
    out = out.permute(0, 2, 3, 1, 4).reshape(b, n * CHUNK, h, dv)[:, :t]
    out = torch.where(live, out, torch.zeros((), device=out.device)).to(q.dtype)
    if not return_state:
        return out
    # the state behind each sequence's last token
    left = (length[:, None] - 1 - pos)
    weight = torch.exp(left.clamp(min=0)[:, None] * log_decay[:, None]) * (left >= 0)[:, None]           # b h t
    kt = torch.where(live, k.to(f), torch.zeros((), device=k.device)).permute(0, 2, 3, 1) * weight[:, :, None]
    vt = torch.where(live, v.to(f), torch.zeros((), device=v.device)).permute(0, 2, 1, 3)
    state = kt.contiguous() @ vt.contiguous()
    if initial_state is not None:
        state = state + torch.exp(length[:, None] * log_decay)[:, :, None, None] * initial_state
    return out, state


def plain_step(q, k, v, log_decay, state, active):
    f = torch.float32
    new = torch.exp(log_decay)[:, None, None] * state + k.to(f)[..., :, None] * v.to(f)[..., None, :]
    out = (q.to(f)[..., :, None] * new).sum(-2)
    if active is not None:
        new = torch.where(active[:, None, None, None], new, state)
        out = torch.where(active[:, None, None], out, torch.zeros((), device=out.device))
    state.copy_(new)
    return out.to(q.dtype)


def plain_top(logits, k, temperature):
    """The k largest of each row in descending order, ties to the lowest class."""
    x = logits.to(torch.float32) + 0.0
    n = x.shape[1]
    bits = x.view(torch.int32)
    order = torch.where(bits >= 0, bits, bits ^ 0x7fffffff).to(torch.int64)                              # as the values are ordered
    key = order * (1 << 32) + (n - 1 - torch.arange(n, device=x.device))
    indices = n - 1 - (torch.topk(key, k, dim=1).values & 0xffffffff)
    values = torch.gather(logits, 1, indices)
    rest = (x / temperature).scatter(1, indices, float('-inf'))
    return values, indices.to(torch.int32), log_sum_exp(rest)


def log_sum_exp(x):
    """-inf for rows that hold nothing but -inf."""
    most = x.amax(1)
    base = torch.where(torch.isfinite(most), most, torch.zeros_like(most))
    return base + torch.log(torch.exp(x - base[:, None]).sum(1))


def plain_distill(logits, values, indices, rest, temperature, weight, grad_loss):
    """(mean over the rows of weight * temperature^2 * KL, its gradient for the logits times grad_loss).

    The unlisted classes join the listed ones as one more class. Where most of the mass is unlisted, both sides' shares of it nearly
    cancel, so what is one value for each listed class is held in 64 bits; the sum over the classes is in 32."""
    n, f = logits.shape[0], torch.float64
    x = logits.to(torch.float32) / temperature
    index = indices.long()
    both = torch.cat([values.to(f) / temperature, rest[:, None].to(f)], 1)
    log_p = both - log_sum_exp(both)[:, None]
    p = torch.exp(log_p)
    base = x.amax(1, keepdim=True)
    e = torch.exp(x - base)
    listed = torch.gather(logits, 1, index).to(f) / temperature - base.to(f)
    unlisted = e.scatter(1, index, 0.0).sum(1, keepdim=True).to(f)
    total = torch.exp(listed).sum(1, keepdim=True) + unlisted
    log_q = torch.cat([listed, torch.log(unlisted)], 1) - torch.log(total)
    row = torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p)).sum(1) * temperature ** 2
    row = torch.where(weight != 0, weight * row, torch.zeros_like(row))
    q = torch.exp(log_q)
    scale = (grad_loss * weight).to(f)[:, None] * (temperature / n)
    share = torch.where(p[:, -1:] > 0, p[:, -1:] / q[:, -1:], torch.zeros_like(total))       # of each unlisted class's q
    grad = e * (scale * (1 - share) / total).to(torch.float32)
    grad.scatter_(1, index, (scale * (q - p)[:, :-1]).to(torch.float32))
    return (row.sum() / n).to(torch.float32), grad.to(logits.dtype)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    size = 4 if case['dtype'] == 'f32' else 2
    if case['op'] == 'attention':
        b, t, h, dk, dv = (case[x] for x in ('batch', 'steps', 'heads', 'dk', 'dv'))
        tokens, states = b * t * h, b * h * dk * dv * 4
        live = tokens * (0.75 if case['ragged'] else 1.0)
        if not case['train']:
            return {'bytes': (live * (2 * dk + dv) + tokens * dv) * size + states * (2 if case['state'] else 0),
                    'flops': 4.0 * live * dk * dv}
        # q, k, v and the gradient of o are read, o and three gradients written
        return {'bytes': (live * 2 * (dk + dv) + tokens * 2 * (dk + dv)) * size + states * (4 if case['state'] else 0),
                'flops': 14.0 * live * dk * dv}
    if case['op'] == 'step':
        b, h, dk, dv = (case[x] for x in ('batch', 'heads', 'dk', 'dv'))
        share = 0.9 if case['active'] else 1.0
        return {'bytes': share * b * h * (8 * dk * dv + (2 * dk + dv) * size) + b * h * dv * size, 'flops': share * 5.0 * b * h * dk * dv}
    n, classes, k = case['rows'], case['classes'], case['k']
    if case['op'] == 'top':
        return {'bytes': n * (classes * size + k * (size + 4) + 4), 'flops': 4.0 * n * classes}
    return {'bytes': n * (2 * classes * size + k * (size + 4) + 8), 'flops': 8.0 * n * classes}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case['op'] == 'attention':
            return exact_attention(s, case)
        if case['op'] == 'step':
            return exact_step(s)
        if case['op'] == 'top':
            return exact_top(s, case)
        return exact_distill(s, case)


def exact_attention(s, case):
    """Token after token: S = decay S + k v^T, o = q S; D = dS/dlog_decay beside it; the gradient R of S backwards."""
    q, k, v = (s[x].detach().double().transpose(0, 1).contiguous() for x in ('q', 'k', 'v'))           # t b h d
    t, b, h, dk = q.shape
    dv = v.shape[-1]
    decay = torch.exp(s['log_decay'].detach().double())[:, None, None]
    length = torch.full((b,), t, device=q.device) if s['lengths'] is None else s['lengths']
    live = (torch.arange(t, device=q.device)[:, None] < length)[:, :, None, None].double()             # t b 1 1
    q, k, v = q * live, k * live, v * live
    ragged, train = s['lengths'] is not None, case['train']
    state = torch.zeros(b, h, dk, dv, device=q.device, dtype=torch.float64)
    if s['initial_state'] is not None:
        state += s['initial_state'].detach()
    slope = torch.zeros_like(state)
    out, gq, gl = torch.empty_like(v), torch.empty_like(q), torch.zeros(b, h, device=q.device, dtype=torch.float64)
    go = s['grad_out'].double().transpose(0, 1).contiguous() * live if train else None
    for i in range(t):
        here = live[i].unsqueeze(-1) > 0
        factor = torch.where(here, decay, 1.0) if ragged else decay
        if train:
            slope = torch.where(here, decay * (slope + state), slope) if ragged else decay * (slope + state)
        state = torch.addcmul(state * factor, k[i].unsqueeze(-1), v[i].unsqueeze(-2))
        torch.matmul(q[i].unsqueeze(-2), state, out=out[i].unsqueeze(-2))
        if train:
            gq[i] = (state @ go[i].unsqueeze(-1)).squeeze(-1)
            gl += (q[i].unsqueeze(-2) @ (slope @ go[i].unsqueeze(-1))).reshape(b, h)
    back = lambda x: x.transpose(0, 1)  # noqa: E731
    if not train:
        return {'out': back(out), 'state': state} if case['state'] else {'out': back(out)}
    grad = torch.zeros_like(state)
    if s['grad_state'] is not None:
        grad += s['grad_state']
        gl += (grad * slope).sum((2, 3))
    gk, gv = torch.empty_like(k), torch.empty_like(v)
    for i in reversed(range(t)):
        grad = torch.addcmul(grad, q[i].unsqueeze(-1), go[i].unsqueeze(-2))
        gk[i] = (grad @ v[i].unsqueeze(-1)).squeeze(-1)
        gv[i] = (k[i].unsqueeze(-2) @ grad).squeeze(-2)
        grad = grad * (torch.where(live[i].unsqueeze(-1) > 0, decay, 1.0) if ragged else decay)
    got = {'out': back(out), 'gq': back(gq * live), 'gk': back(gk * live), 'gv': back(gv * live), 'glog_decay': gl.sum(0)}
    if s['initial_state'] is not None:
        got.update(state=state, ginitial_state=grad)
    return got


def exact_step(s):
    q, k, v, state = (s[x].double() for x in ('q', 'k', 'v', 'state'))
    new = torch.exp(s['log_decay'].double())[None, :, None, None] * state + torch.einsum('bhi,bhj->bhij', k, v)
    out = torch.einsum('bhi,bhij->bhj', q, new)
    if s['active'] is not None:
        idle = ~s['active']
        new[idle], out[idle] = state[idle], 0.0
    return {'out': out, 'state': new}


def exact_top(s, case):
    """By a stable sort; the rest by setting aside what it puts first."""
    parts = []
    for x in s['logits'].split(max(1, (1 << 26) // case['classes'])):
        x = x.double()
        value, index = torch.sort(x, dim=1, descending=True, stable=True)
        left = torch.nn.functional.pad(value[:, case['k']:], (0, 1), value=float('-inf'))               # k may be all of them
        rest = torch.logsumexp(left / case['temperature'], 1)
        parts.append((value[:, :case['k']].clone(), index[:, :case['k']].int(), rest))
    return dict(zip(('values', 'indices', 'rest'), (torch.cat(p) for p in zip(*parts))))


def exact_distill(s, case):
    n, tau, loss, grads = case['rows'], case['temperature'], 0.0, []
    scale = s['grad_loss'].double()
    for a in range(0, n, max(1, (1 << 26) // case['classes'])):
        e = min(n, a + max(1, (1 << 26) // case['classes']))
        x, w = s['logits'].detach()[a:e].double() / tau, s['weight'][a:e].double()
        index = s['indices'][a:e].long()
        teacher = torch.softmax(torch.cat([s['values'][a:e].double() / tau, s['rest'][a:e, None].double()], 1), 1)
        listed_mass, rest_mass = teacher[:, :-1], teacher[:, -1]
        student = torch.softmax(x, 1)
        away = torch.ones_like(student, dtype=torch.bool).scatter_(1, index, False)
        rest_student = (student * away).sum(1)
        kl = torch.xlogy(listed_mass, listed_mass).sum(1) - (listed_mass * torch.log_softmax(x, 1).gather(1, index)).sum(1)
        kl += torch.where(rest_mass > 0, rest_mass * (rest_mass.log() - rest_student.log()), torch.zeros_like(kl))
        loss += float((w * kl).sum()) * tau ** 2 / n
        target = student * away * torch.where(rest_mass > 0, rest_mass / rest_student, torch.zeros_like(kl))[:, None]
        target.scatter_(1, index, listed_mass)
        grads.append((student - target) * (scale * w * tau / n)[:, None])
    return {'loss': torch.tensor(loss, dtype=torch.float64), 'grad': torch.cat(grads)}
