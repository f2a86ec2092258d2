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


@pytest.mark.parametrize('by_slots', [False, True])
def test_rows_without_an_event_leave_their_user(by_slots):
    """token_type 0 is padding, to a step as to predict: the row's user keeps states and
    position, the others get what a step of their own gives them, and the next event follows
    predict on the history without the row."""
    m, batch, _ = make(B=4)
    m.eval()
    seq, tt, feat = batch[0], batch[3].clone(), batch[6]
    T = seq.shape[1]
    head, last = slice(0, T - 1), slice(T - 1, T)
    _, s = m.stream_begin(seq[:, head], to_rows(feat, head), tt[:, head])
    kept, was = [x.clone() for x in s.states], s.position.clone()
    kind = tt[:, -1].clone()
    assert bool((kind > 0).all())
    kind[1] = kind[3] = 0
    order = torch.arange(4, device=DEV) if by_slots else None
    got = m.stream_step(s, seq[:, -1], to_rows(feat, last), kind, order)
    want = m.predict(seq, feat, tt)
    for u in range(4):
        if kind[u] == 0:
            assert all(torch.equal(x[u], k[u]) for x, k in zip(s.states, kept)) and s.position[u] == was[u]
        else:
            assert nrel(got[u], want[u]) < TOL and s.position[u] == was[u] + 1
    late = torch.tensor([1, 3], device=DEV)
    got = m.stream_step(s, seq[late, -1], {k: v[late, -1:] for k, v in feat.items()}, tt[late, -1], late)
    assert nrel(got, want[late]) < TOL
    s.check()


def test_padding_between_the_events_of_one_user():
    m, batch, _ = make(B=2)
    m.eval()
    seq, tt, feat = batch[0], batch[3], batch[6]
    T = seq.shape[1]
    head = slice(0, T - 2)
    _, a = m.stream_begin(seq[:, head], to_rows(feat, head), tt[:, head])
    _, b = m.stream_begin(seq[:, head], to_rows(feat, head), tt[:, head])
    at = torch.tensor([T - 2, T - 1], device=DEV)
    user = torch.zeros(2, dtype=torch.int64, device=DEV)
    want = m.stream_step(a, seq[user, at], {k: v[user, at][:, None] for k, v in feat.items()}, tt[user, at], user)
    at, user = torch.tensor([T - 2, T - 2, T - 1], device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    kind = tt[user, at].clone()
    kind[1] = 0
    got = m.stream_step(b, seq[user, at], {k: v[user, at][:, None] for k, v in feat.items()}, kind, user)
    assert nrel(got[[0, 2]], want) < TOL and a.position.tolist() == b.position.tolist() == [T, T - 2]
    for x, y in zip(a.states, b.states):
        assert nrel(x, y) < TOL
    # a slot outside the stream is named all the same
    m.stream_step(b, seq[:1, 0], {k: v[:1, :1] for k, v in feat.items()}, torch.zeros_like(tt[:1, 0]),
                  torch.tensor([7], device=DEV))
    with pytest.raises(ValueError):
        b.check()


def test_token_types_of_another_count_are_refused():
    m, batch, _ = make(B=2)
    m.eval()
    seq, tt, feat = batch[0], batch[3], batch[6]
    _, s = m.stream_begin(seq, feat, tt)
    was = s.position.tolist()
    with pytest.raises(ValueError):
        m.stream_step(s, seq[:, 0], to_rows(feat, slice(0, 1)), tt[:1, 0])
    assert s.position.tolist() == was


@pytest.mark.parametrize('n,pool', [(1, 1), (7, 3), (256, 40), (257, 40), (5000, 1), (5000, 300), (70001, 2 ** 17 - 1),
                                    (70001, 2 ** 31 - 1)])
def test_earlier_events_of_a_slot(n, pool):
    """Counted without an n^2 buffer: 200 bytes an event at most beside the sort's own counts
    (8 KB for 1024 events)."""
    from tencent_recommendation_2025_amd.model import _earlier_of_slot
    g = torch.Generator(device=DEV).manual_seed(n)
    slots = torch.randint(0, pool, (n,), generator=g, device=DEV)
    slots[torch.rand(n, generator=g, device=DEV) < 0.1] = pool
    seen, want = {}, []
    for s in slots.tolist():
        want.append(seen.get(s, 0))
        seen[s] = want[-1] + 1
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = _earlier_of_slot(slots, pool)
    assert got.dtype == torch.int64 and got.tolist() == want
    assert torch.cuda.max_memory_allocated() - before < 210 * n + (1 << 20)


def test_many_events_in_one_step():
    """900 events of 6 users in one call, in a graph too: the users' states are those of 150
    calls, and every replay has the eager call's."""
    m, batch, _ = make(B=6)
    m.eval()
    seq, tt, feat = batch[0], batch[3], batch[6]
    T = seq.shape[1]
    cut, turns = T - 5, 150
    head = slice(0, cut)
    first = lambda: m.stream_begin(seq[:, head], to_rows(feat, head), tt[:, head])[1]  # noqa: E731
    one, all_, kept = first(), first(), first()
    g = torch.Generator(device=DEV).manual_seed(7)
    at = torch.randint(cut, T, (turns, 6), generator=g, device=DEV)
    user = torch.stack([torch.randperm(6, generator=g, device=DEV) for _ in range(turns)])
    rows = lambda u, t: {k: v[u, t][:, None] for k, v in feat.items()}  # noqa: E731
    want = torch.cat([m.stream_step(one, seq[u, t], rows(u, t), tt[u, t], u) for u, t in zip(user, at)])
    user, at = user.reshape(-1), at.reshape(-1)
    args = seq[user, at], rows(user, at), tt[user, at], user
    got = m.stream_step(all_, *args)
    # 150 events more pass through the states than in one call of 6: sums of 150 more terms
    tol = 2 * TOL
    assert nrel(got, want) < tol and all_.position.tolist() == one.position.tolist() == [cut + turns] * 6
    for x, y in zip(all_.states, one.states):
        assert nrel(x, y) < tol
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.stream_step(kept, *args)
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = m.stream_step(kept, *args)
    for _ in range(3):
        gr.replay()
        torch.cuda.synchronize()
        again = m.stream_step(all_, *args)
        torch.cuda.synchronize()
        assert torch.equal(out, again) and torch.equal(kept.position, all_.position)
        for x, y in zip(kept.states, all_.states):
            assert torch.equal(x, y)


def test_slots_that_are_no_numbers_of_slots_are_refused():
    """A mask would be read as slots 0 and 1."""
    m, batch, _ = make(B=2)
    m.eval()
    seq, tt, feat = batch[0], batch[3], batch[6]
    _, s = m.stream_begin(seq, feat, tt)
    was = s.position.tolist()
    for slots in (torch.tensor([True, False], device=DEV), torch.tensor([0.0, 1.0], device=DEV)):
        with pytest.raises(ValueError):
            m.stream_step(s, seq[:, 0], to_rows(feat, slice(0, 1)), tt[:, 0], slots)
    assert s.position.tolist() == was
    m.stream_step(s, seq[:, -1], to_rows(feat, slice(seq.shape[1] - 1, None)), tt[:, -1],
                  torch.tensor([1, 0], dtype=torch.int16))
    assert s.position.tolist() == [w + 1 for w in was]
