"""CPU checks of the decay block's operators: every refusal of the C entry points comes
before a launch, the Python wrappers refuse what the kernels do not take, and the rotary
frequencies are the formulas'."""
import ctypes as C
import math

import pytest
import torch

from tencent_recommendation_2025_amd import _lib as L
from tencent_recommendation_2025_amd import functional as G
from tencent_recommendation_2025_amd import kernels as K


@pytest.fixture(scope='module')
def lib():
    return L.lib()


def err(lib):
    return lib.grk_last_error().decode()


P = 4096   # a pointer that no call here reaches


def test_rotary_refusals(lib):
    def call(dtype=L.GRK_BF16, itype=L.GRK_I64, rows=4, heads=2, hd=64, rd=64, ldx=128, ldy=128, x=P, y=2 * P,
             pos=P, freqs=P):
        return lib.grk_rotary(x, ldx, y, ldy, dtype, pos, itype, freqs, rows, heads, hd, rd, 0, 1.0, 0, None)

    for kw, word in ((dict(dtype=7), 'dtype'), (dict(itype=5), 'int32 or int64'), (dict(rows=-1), 'rows'),
                     (dict(heads=0), 'heads'), (dict(hd=0), 'head_dim'), (dict(rd=3), 'rotary_dim'),
                     (dict(rd=66), 'rotary_dim'), (dict(rd=0), 'rotary_dim'), (dict(ldx=127), 'strides'),
                     (dict(x=None), 'required'), (dict(freqs=None), 'required'), (dict(y=P, ldy=256), 'in place'),
                     (dict(heads=1 << 20, hd=64), '2^20')):
        assert call(**kw) == L.GRK_EINVAL and word in err(lib), (kw, err(lib))
    assert call(rows=0, x=None, y=None) == L.GRK_OK


def args(**kw):
    a = dict(batch=2, heads=2, seq_len=5, head_dim=64, dtype=L.GRK_BF16, scale=1.0, q=P, k=P, v=P, ldq=128, ldk=128,
             ldv=128, log_decay=P, key_valid=None, seq_range=None, row_base=None, num_rows=None, capacity=0)
    a.update(kw)
    return L.GrkDecayArgs(*[a[n] for n, _ in L.GrkDecayArgs._fields_])


def test_decay_attn_refusals(lib):
    fwd = lambda a, out=P, ldo=128: lib.grk_decay_attn_fwd(a, None, None, out, ldo, None, 0, None)  # noqa: E731
    bwd = lambda a, g=P: lib.grk_decay_attn_bwd(a, g, 128, P, 128, P, 128, P, 128, None, 0, None)  # noqa: E731
    for kw, word in ((dict(dtype=9), 'dtype'), (dict(batch=-1), 'batch'), (dict(heads=0), 'heads'),
                     (dict(seq_len=-1), 'seq_len'), (dict(q=None), 'q required'), (dict(ldk=127), 'k: row stride'),
                     (dict(log_decay=None), 'log_decay'), (dict(row_base=P), 'seq_range'),
                     (dict(batch=1 << 21), '2^21'), (dict(batch=0, row_base=P, seq_range=P, capacity=3), 'capacity')):
        for f in (fwd, bwd):
            if 'row_base' in kw and 'capacity' not in kw:
                kw = dict(kw, capacity=10)
            assert f(args(**kw)) == L.GRK_EINVAL and word in err(lib), (kw, err(lib))
    assert fwd(args(head_dim=129, ldq=300, ldk=300, ldv=300)) == L.GRK_EUNSUPPORTED and '128' in err(lib)
    assert fwd(args(), out=None) == L.GRK_EINVAL and bwd(args(), g=None) == L.GRK_EINVAL
    # a long sequence of one head is cut into segments: their states need a workspace
    long = args(batch=1, heads=1, seq_len=100_000, ldq=64, ldk=64, ldv=64)
    assert lib.grk_decay_attn_workspace(long, 0) > 0
    assert fwd(long, ldo=64) == L.GRK_EINVAL and 'workspace' in err(lib)
    assert fwd(args(batch=0)) == L.GRK_OK and fwd(args(seq_len=0)) == L.GRK_OK


def test_decay_step_refusals(lib):
    def call(n=3, heads=2, hd=64, dtype=L.GRK_F32, itype=L.GRK_I64, ld=128, slots=None, num=3, q=P, state=P, ws=0):
        return lib.grk_decay_attn_step(q, ld, P, ld, P, ld, dtype, P, n, heads, hd, 1.0, state, num, slots, itype,
                                       None, P, ld, None, ws, None)

    for kw, word in ((dict(dtype=5), 'dtype'), (dict(itype=7), 'slots'), (dict(n=-1), 'n >= 0'),
                     (dict(ld=127), 'row strides'), (dict(num=2), 'num_slots'), (dict(q=None), 'required'),
                     (dict(n=300, num=500, slots=P), 'workspace'), (dict(n=1 << 24, num=1 << 24), '2^24')):
        assert call(**kw) == L.GRK_EINVAL and word in err(lib), (kw, err(lib))
    assert call(hd=200, ld=400) == L.GRK_EUNSUPPORTED
    assert call(n=0) == L.GRK_OK


def test_head_norm_refusals(lib):
    def fwd(rows=4, heads=2, hd=64, dtype=L.GRK_F32, ldx=128, x=P, y=P, eps=1e-5, gate=None, ldg=0):
        return lib.grk_head_norm_fwd(x, ldx, gate, ldg, P, P, eps, rows, heads, hd, dtype, y, 128, None)

    for kw, word in ((dict(dtype=4), 'dtype'), (dict(hd=2049, ldx=5000), 'head_dim'), (dict(rows=-2), 'rows'),
                     (dict(ldx=100), 'x: row stride'), (dict(x=None), 'x required'), (dict(y=None), 'y required'),
                     (dict(eps=-1.0), 'eps'), (dict(gate=P, ldg=5), 'gate: row stride')):
        assert fwd(**kw) == L.GRK_EINVAL and word in err(lib), (kw, err(lib))
    assert lib.grk_head_norm_bwd(P, 128, P, 128, None, 0, P, P, 1e-5, 4, 2, 64, L.GRK_F32, P, 128, None, 0, P, P,
                                 None, 0, None) == L.GRK_EINVAL and 'workspace' in err(lib)
    assert lib.grk_head_norm_bwd(P, 128, P, 128, P, 128, P, P, 1e-5, 4, 2, 64, L.GRK_F32, P, 128, None, 0, None, None,
                                 None, 0, None) == L.GRK_EINVAL and 'dgate' in err(lib)


def test_wrappers_refuse_host_tensors():
    x = torch.zeros(4, 128)
    pos, f = torch.zeros(4, dtype=torch.int64), torch.ones(32, dtype=torch.float64)
    lg = torch.zeros(2)
    with pytest.raises(L.GrkError, match='device'):
        K.rotary(x, pos, f, 2)
    with pytest.raises(L.GrkError, match='device'):
        K.decay_attn_fwd(x, x, x, lg, 1, 4)
    with pytest.raises(L.GrkError, match='device'):
        K.decay_attn_step(x, x, x, lg, torch.zeros(4, 2, 64, 64))
    with pytest.raises(L.GrkError, match='device'):
        K.head_norm_fwd(x, None, None, 2)


def test_learned_decays_and_freqs_are_refused():
    x = torch.zeros(4, 128)
    with pytest.raises(L.GrkError, match='log_decay'):
        G.decay_attn(torch.zeros(4, 384), torch.zeros(2, requires_grad=True), 1, 4)
    with pytest.raises(L.GrkError, match='freqs'):
        G.rotary(x, torch.zeros(4, dtype=torch.int64), torch.ones(32, dtype=torch.float64, requires_grad=True), 2)
    with pytest.raises(L.GrkError, match='gate'):
        G.head_norm(x, None, None, 2, gate=x[:2])


def test_overlap_of_views():
    buf = torch.zeros(8, 64)
    a, b = buf[:, :32], buf[:, 32:]
    assert not K._overlap(a, b) and not K._overlap(b, a)
    assert K._overlap(buf[:, :33], b) and K._overlap(b, buf[:, :33])
    assert K._overlap(a, a) and K._overlap(a, buf[2:, :32]) and not K._overlap(buf[:4], buf[4:])
    assert K._overlap(a, buf.view(16, 32)) and not K._overlap(a, torch.zeros(8, 32))
    assert not K._overlap(b[1:], a) and K._overlap(buf[:, 16:48], b)


def test_ranges_that_meet():
    buf = torch.zeros(4, 2, 8, 8)
    assert K._meet(buf, buf) and K._meet(buf[:3], buf[1:]) and not K._meet(buf[:2], buf[2:])
    rows = buf.view(16, 32)
    assert K._meet(rows[:, 16:], buf[3:]) and not K._meet(rows[:4, :16], buf[1:])
    assert not K._meet(buf[:0], buf) and not K._meet(torch.zeros(4), buf)
    # what is no matrix is refused by its shape, not compared
    assert not K._overlap(torch.zeros(8), rows) and not K._overlap(rows, buf)


def test_layers_refuse_columns_that_they_cannot_split():
    pos, f = torch.zeros(4, dtype=torch.int64), torch.ones(4, dtype=torch.float64)
    for cols in (100, 3 * 65):
        with pytest.raises(L.GrkError, match='side by side'):
            G.rotary_qk(torch.zeros(4, cols), pos, f, 2)
    with pytest.raises(L.GrkError, match='freqs'):
        G.rotary_qk(torch.zeros(4, 96), pos, f.clone().requires_grad_(True), 2)
    w, lg = torch.ones(16), torch.zeros(2)
    with pytest.raises(L.GrkError, match='side by side'):
        G.decay_core(torch.zeros(4, 66), lg, w, w, 1, 4)
    with pytest.raises(L.GrkError, match='side by side'):
        G.decay_core(torch.zeros(4, 64), lg, w, None, 1, 4)
    with pytest.raises(L.GrkError, match='log_decay'):
        G.decay_core(torch.zeros(4, 64), lg.clone().requires_grad_(True), w, w, 1, 4)


def test_rotary_frequencies():
    f, s = K.rotary_frequencies(8)
    assert f.dtype == torch.float64 and s == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    lin, s = K.rotary_frequencies(8, scaling={'kind': 'linear', 'factor': 4})
    assert torch.equal(lin, f / 4) and s == 1.0
    base, _ = K.rotary_frequencies(8, scaling={'kind': 'base', 'factor': 4})
    assert base[0] == 1.0 and math.isclose(float(base[-1]), float(f[-1]) / 4, rel_tol=1e-12)
    part, s = K.rotary_frequencies(64, scaling={'kind': 'by_parts', 'factor': 8, 'window': 4096})
    plain, _ = K.rotary_frequencies(64)
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(part[turns >= 32], plain[turns >= 32])
    assert torch.allclose(part[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15) and bool((turns <= 1).any())
    mid = (turns > 1) & (turns < 32)
    assert bool((part[mid] < plain[mid]).all() and (part[mid] > plain[mid] / 8).all())
    assert math.isclose(s, 0.1 * math.log(8) + 1)
    for bad in ({'kind': 'spline', 'factor': 2}, {'kind': 'linear'}, {'kind': 'linear', 'factor': 0.5}, {'factor': 2},
                {'kind': 'by_parts', 'factor': 2, 'window': 0}):
        with pytest.raises((ValueError, KeyError)):
            K.rotary_frequencies(8, scaling=bad)
    with pytest.raises(ValueError):
        K.rotary_frequencies(7)


def test_args_struct_matches_header():
    """ctypes lays grk_decay_args out as the C compiler does: 6 4-byte fields, then 8-byte ones."""
    a = L.GrkDecayArgs
    assert a.q.offset == 24 and a.ldq.offset == 48 and a.log_decay.offset == 72 and a.capacity.offset == 112
    assert C.sizeof(a) == 120
