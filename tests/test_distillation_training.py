"""Training by a teacher: poreplex_amd/training.py with torch_ops (the shipped classifier's answers as targets, the decay recurrence
as a layer).  CPU legs: what does not need the kernels; -m gpu legs: the layer against its plain statement, one step after the other,
gradients, a whole training run."""
import numpy as np
import pytest

torch = pytest.importorskip('torch')
torch.set_num_threads(2)

from poreplex_amd import torch_ops as ops  # noqa: E402
from poreplex_amd import training as TR  # noqa: E402
from poreplex_amd.torch_models import DemuxNet  # noqa: E402

gpu = pytest.mark.gpu


def test_default_classifier_is_what_it_was():
    torch.manual_seed(3)
    model = TR.DemuxClassifier()
    torch.manual_seed(3)
    parts = [TR._KerasLSTM(1, 48), TR._KerasLSTM(1, 48), TR._KerasLSTM(96, 64), torch.nn.Linear(64, 5)]
    want = [p for m in parts for p in m.parameters()]
    assert len(list(model.parameters())) == len(want) and all(torch.equal(a, b) for a, b in zip(model.parameters(), want))
    assert set(DemuxNet().state_dict()) == {'{}.{}_l0'.format(m, n) for m in ('fwd', 'bwd', 'top')
                                            for n in ('weight_ih', 'weight_hh', 'bias_ih', 'bias_hh')}


def test_refusals(tmp_path):
    with pytest.raises(ValueError, match='lstm'):
        TR.DemuxClassifier(top='gru')
    with pytest.raises(ValueError, match='heads'):
        TR.DecayRecurrence(8, 10, heads=4)
    with pytest.raises(ValueError, match='cannot be exported'):
        TR.export_demux_bundle(TR.DemuxClassifier(top='decay'), str(tmp_path / 'x.npz'), np.zeros(3))
    with pytest.raises(ValueError, match='on a GPU only'):
        TR.DemuxClassifier(top='decay')(torch.zeros(2, 300))


def test_no_samples_and_no_answers_are_refused():
    with pytest.raises(ValueError, match='no samples'):
        TR.distillation_targets(TR.DemuxClassifier(), torch.zeros(0, 300), device='cpu')
    with pytest.raises(ValueError, match='no answers'):
        ops.TopLogits.cat([])


def test_the_teachers_modes_come_back(monkeypatch):
    monkeypatch.setattr(ops, 'top_logits', lambda x, k, tau: ops.TopLogits(x[:, :k], torch.arange(k).repeat(len(x), 1), x[:, -1], tau))
    teacher = TR.DemuxClassifier().train()
    teacher.drop1.eval()
    modes, x = [m.training for m in teacher.modules()], torch.randn(7, 300)
    first = TR.distillation_targets(teacher, x, device='cpu', batch_size=4)
    assert [m.training for m in teacher.modules()] == modes and len(first) == 7
    assert first.values.equal(TR.distillation_targets(teacher, x, device='cpu').values)          # in evaluation mode: no dropout
    with pytest.raises(ValueError, match='LSTM'):
        TR.distillation_targets(teacher, x[:, :, None, None], device='cpu')
    assert [m.training for m in teacher.modules()] == modes


def test_trainer_takes_top_logits(tmp_path):
    """Targets that are TopLogits go through the trainer's split, shuffling and batches like labels: every sample meets its own."""
    n = 70
    x = torch.arange(float(n))[:, None].repeat(1, 4)
    y = ops.TopLogits(x[:, :2].clone(), torch.arange(n)[:, None].repeat(1, 2), torch.arange(float(n)), 2.0)

    def loss(out, t):
        assert t.temperature == 2.0 and len(t) == len(out)
        assert torch.equal(t.values[:, 0], out.detach()[:, 0].round()) and torch.equal(t.rest, t.values[:, 0])
        return (out - out.detach()).square().mean() + 1.0

    class Same(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.zero = torch.nn.Parameter(torch.zeros(1))

        def forward(self, v):
            return v + self.zero
    hist = TR.Trainer(Same(), loss, batch_size=16, epochs=2, validation_split=0.2, output_dir=str(tmp_path)).fit(x, y)
    assert len(hist) == 2 and hist[0]['loss'] == 1.0


def plain_layer(layer, x, lengths=None):
    """64 bits, step after step"""
    w = {n: p.detach().double().cpu() for n, p in layer.named_parameters()}
    x = x.double().cpu()
    q, k, v = (x @ w['qkv.weight'].T + w['qkv.bias']).unflatten(-1, (3, layer.heads, layer.width)).unbind(-3)
    a = torch.exp(-torch.exp(w['rate']))[:, None, None]
    state, rows = torch.zeros(len(x), layer.heads, layer.width, layer.width, dtype=torch.float64), []
    for t in range(x.shape[1]):
        live = torch.ones(len(x), 1, 1, 1, dtype=torch.bool) if lengths is None else (t < lengths)[:, None, None, None]
        state = torch.where(live, a * state + k[:, t, :, :, None] * v[:, t, :, None, :], state)
        rows.append(torch.where(live[..., 0], (q[:, t, :, None] @ state)[..., 0, :] * layer.width ** -0.5, torch.zeros((), dtype=torch.float64)))
    return torch.stack(rows, 1).flatten(-2) @ w['out.weight'].T + w['out.bias'], state


@gpu
def test_layer_and_its_steps():
    """float32: products of 96 and 64 terms around the recurrence (2^-24 * 160 of the absolute terms, some hundred times the values)"""
    torch.manual_seed(1)
    layer = TR.DecayRecurrence(96, 64).cuda()
    x, lengths = torch.randn(5, 75, 96, device='cuda'), torch.tensor([75, 0, 1, 33, 64])
    want, want_state = plain_layer(layer, x, lengths)
    with torch.no_grad():
        out, state = layer(x, lengths.cuda())
    room = 2.0 ** -24 * 160 * 100
    assert float((out.double().cpu() - want).abs().max()) <= room and float((state.double().cpu() - want_state).abs().max()) <= room
    streams, rows = layer.new_state(5), []
    for t in range(75):
        rows.append(layer.step(x[:, t], streams, (t < lengths).cuda()))
    assert float((torch.stack(rows, 1).double().cpu() - want).abs().max()) <= room
    assert float((streams.double().cpu() - want_state).abs().max()) <= room
    # a window in two pieces, the state carried between them
    with torch.no_grad():
        first, middle = layer(x[:, :31])
        second, last = layer(x[:, 31:], state=middle)
        whole, end = layer(x)
    assert float((torch.cat([first, second], 1) - whole).abs().max()) <= 2 * room and float((last - end).abs().max()) <= 2 * room


@gpu
def test_student_of_the_shipped_classifier():
    """the shipped classifier's answers, a student with a decay recurrence: the trainer runs, and one batch's gradients are those of
    the plain formula (float32 autograd through LSTM layers on both sides: 1e-4 of each gradient's norm)"""
    torch.manual_seed(2)
    x, _ = TR.synthetic_demux_dataset(300, seed=4)
    teacher = DemuxNet()
    targets = TR.distillation_targets(teacher, x, k=3, temperature=2.0)
    assert len(targets) == 300 and targets.values.device.type == 'cpu' and targets.temperature == 2.0
    log_p = teacher(x.cuda()).cpu()
    top = torch.sort(log_p, dim=1, descending=True, stable=True)
    assert torch.equal(targets.indices.long(), top.indices[:, :3]) and torch.equal(targets.values, top.values[:, :3])
    model = TR.DemuxClassifier(noise=0.0, drop1=0.0, drop2=0.0, top='decay')
    hist = TR.Trainer(model, ops.distillation_loss, device='cuda', batch_size=64, epochs=2).fit(x, targets)
    assert len(hist) == 2 and all(np.isfinite(h['loss']) and np.isfinite(h['val_loss']) for h in hist)
    model.train()
    batch, t = x[:40].cuda(), targets[:40].to('cuda')
    params = [p for p in model.parameters() if p.requires_grad]
    got = torch.autograd.grad(ops.distillation_loss(model(batch), t), params)
    log_q = torch.log_softmax(model(batch).double() / 2.0, 1)
    both = torch.log_softmax(torch.cat([t.values.double() / 2.0, t.rest.double()[:, None]], 1), 1)
    away = torch.ones_like(log_q, dtype=torch.bool).scatter_(1, t.indices.long(), False)
    student = torch.cat([log_q.gather(1, t.indices.long()), log_q.masked_fill(~away, -float('inf')).logsumexp(1, keepdim=True)], 1)
    want = torch.autograd.grad(4.0 * (both.exp() * (both - student)).sum(1).mean(), params)
    for a, b in zip(got, want):
        assert float((a - b).norm()) <= 1e-4 * float(b.norm()) + 1e-9
