"""The decay block in serving: predict and streams under inference mode beside training,
rows of a step that hold no event, and steps of many events.

Tolerances as in test_gpu_decay_model: a model's fp32 layers 2 * 2000 * 2^-24, normwise."""
import pytest
import torch
import torch.nn.functional as F

from test_gpu_decay_model import DEV, make, nrel, to_rows

pytestmark = pytest.mark.gpu
TOL = 2 * 2000 * 2.0 ** -24


def gradients(m, batch):
    m.train()
    m.zero_grad()
    pos, neg = m(*batch[:9])
    ntt = batch[4] == 1
    (F.softplus(-pos[ntt]).mean() + F.softplus(neg[ntt]).mean()).backward()
    return {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}


@pytest.mark.parametrize('block,rotary', [('decay', True), ('decay', None), ('softmax', True), ('softmax', None),
                                          ('hstu', None)])
def test_training_after_predict_under_inference_mode(block, rotary):
    """What the first predict leaves behind (frequencies, constants) may be saved for a
    backward later on: the gradients are those of a model that never served."""
    from tencent_recommendation_2025_amd import model as M
    m, batch, _ = make(block, rotary)
    want = gradients(make(block, rotary)[0], batch)
    M._UNIT_ROWS.clear()
    m.eval()
    with torch.inference_mode():
        assert bool(torch.isfinite(m.predict(batch[0], batch[6], batch[3])).all())
    got = gradients(m, batch)
    assert set(got) == set(want)
    for n in want:
        if not n.endswith('k_linear.bias'):   # (softmax scores do not change with it: rounding alone)
            assert nrel(got[n], want[n]) < 100 * TOL, n


def test_trainer_after_predict_under_inference_mode():
    from tencent_recommendation_2025_amd import model as M
    from tencent_recommendation_2025_amd.optim import FusedAdamW
    from tencent_recommendation_2025_amd.train import Trainer
    losses = []
    for serve in (False, True):
        m, batch, _ = make(hidden=128)
        tr = Trainer(m, FusedAdamW(m, lr=1e-3), loss='bce')
        M._UNIT_ROWS.clear()
        if serve:
            m.eval()
            with torch.inference_mode():
                m.predict(batch[0], batch[6], batch[3])
            m.train()
        losses.append(torch.stack([tr.step(batch).clone() for _ in range(3)]))
    assert torch.equal(*losses)


def test_a_stream_begun_under_inference_mode_goes_on_outside():
    m, batch, _ = make(B=3)
    m.eval()
    seq, tt, feat = batch[0], batch[3], batch[6]
    T = seq.shape[1]
    head, last = slice(0, T - 1), slice(T - 1, T)
    _, plain = m.stream_begin(seq[:, head], to_rows(feat, head), tt[:, head])
    want = m.stream_step(plain, seq[:, -1], to_rows(feat, last), tt[:, -1])
    with torch.inference_mode():
        first, stream = m.stream_begin(seq[:, head], to_rows(feat, head), tt[:, head], slots=4)
    got = m.stream_step(stream, seq[:, -1], to_rows(feat, last), tt[:, -1], torch.arange(3, device=DEV))
    assert nrel(got, want) < TOL and stream.position.tolist() == [T, T, T, 0]
    stream.place(torch.tensor([3, 1, 0], device=DEV), plain)
    stream.clear(torch.tensor([2], device=DEV))
    assert stream.position.tolist() == [T, T, 0, T] and torch.equal(stream.states[0][3], plain.states[0][0])
    stream.check()
    with torch.inference_mode():   # and back under it
        m.stream_step(stream, seq[:1, -1], to_rows({k: v[:1] for k, v in feat.items()}, last), tt[:1, -1],
                      torch.tensor([2], device=DEV))
    assert stream.position.tolist() == [T, T, 1, T]
