"""GPU parity of the decay block's operators (rotary positions, decayed linear attention,
the per-head norm) against plain 64-bit references.

Tolerances.  u = eps / 2 of the row type is one rounding of the output.
* rotary: cos and sin are off by at most 8 * 2^-24 (the fp32 fraction of a turn: pi 2^-24;
  sincospif 2 ulp; the scale's rounding), products and sum by 3 * 2^-24 more:
  |err| <= u |y| + 12 * 2^-24 scale (|x_i| + |x_j|), element by element.
* decayed attention: u for the output's rounding, and for bf16 rows u for the rounding of
  the score matrix and u for that of the state as operands (independent roundings of the
  terms of a sum of independent terms: normwise at most u each); fp32 sums of at most
  head_dim + 64 + T / 64 terms at 2^-24 each, and the powers of g (argument up to 20:
  20 * 2^-24): tol = u (fp32, fp16) or 3 u (bf16), plus 300 * 2^-24, in the 2-norm.  A
  row's own error may exceed the whole's: 8 times that of the rows' common size.
* head norm: statistics and affine are about 20 fp32 roundings, amplified by at most
  1 + |mean| / std = 16 in the test data; the 16-bit types' hardware exponential adds
  2^-21: tol = u + 320 * 2^-24 (2-norm); the weight gradients are fp32 sums of rows.
"""
import math
import zlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
DT = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}


@pytest.fixture(scope='module')
def K():
    from tencent_recommendation_2025_amd import _lib, kernels
    _lib.lib()
    return kernels


@pytest.fixture(scope='module')
def G():
    from tencent_recommendation_2025_amd import functional
    return functional


def gen(*key):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(key).encode()))


def randn(g, *shape, dt=torch.float32):
    return torch.randn(*shape, device=DEV, generator=g).to(dt)


def u_of(dt):
    return torch.finfo(dt).eps / 2


def close(got, want, tol, rows=True):
    got, want = got.double(), want.double()
    assert got.shape == want.shape and bool(torch.isfinite(got).all())
    err, size = (got - want).norm(), want.norm()
    assert err <= tol * size + 1e-30, f'2-norm {float(err / size):.3e} > {tol:.3e}'
    if rows and got.dim() == 2 and got.shape[0] > 1:
        common = size / math.sqrt(want.shape[0])
        worst = (got - want).norm(dim=1) / torch.maximum(want.norm(dim=1), common).clamp(min=1e-30)   # all of it 0
        assert worst.max() <= 8 * tol, f'row {int(worst.argmax())}: {float(worst.max()):.3e}'


# ------------------------------------------------------------------ rotary ----
def rotary_ref(x, pos, freqs, heads, layout, scale, sign=1.0):
    N, D = x.shape
    r = freqs.numel()
    z = x.double().view(N, heads, D // heads).clone()
    ang = pos.double()[:, None] * freqs
    c, s = (torch.cos(ang) * scale)[:, None], (sign * torch.sin(ang) * scale)[:, None]
    a, b = (z[..., :r], z[..., r:2 * r]) if layout == 'half' else (z[..., 0:2 * r:2], z[..., 1:2 * r:2])
    ya, yb = a * c - b * s, b * c + a * s
    room = torch.zeros_like(z)
    lim = 12 * 2.0 ** -24 * scale * (a.abs() + b.abs())
    if layout == 'half':
        z[..., :r], z[..., r:2 * r] = ya, yb
        room[..., :r] = room[..., r:2 * r] = lim
    else:
        z[..., 0:2 * r:2], z[..., 1:2 * r:2] = ya, yb
        room[..., 0:2 * r:2] = room[..., 1:2 * r:2] = lim
    return z.view(N, D), room.view(N, D)


def rotary_close(got, ref, dt):
    want, room = ref
    # fp16's smallest steps are 2^-25 apart from rounding
    bad = (got.double() - want).abs() > u_of(dt) * want.abs() + room + (2.0 ** -25 if dt == torch.float16 else 0)
    assert not bool(bad.any()), f'{int(bad.sum())} elements'


@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('dt', list(DT))
@pytest.mark.parametrize('rows,heads,hd,rd,far', [(1, 1, 2, 2, 5), (3, 2, 16, 16, 300), (65, 3, 20, 6, 1000),
                                                  (129, 16, 64, 64, 2_000_000), (2050, 8, 80, 32, 40_000),
                                                  (7, 1, 129, 128, 77), (40, 2, 512, 512, 9999)])
def test_rotary(K, layout, dt, rows, heads, hd, rd, far):
    dt = DT[dt]
    g = gen('rot', rows, hd)
    x = randn(g, rows, heads * hd, dt=dt)
    pos = torch.randint(-far, far, (rows,), generator=g, device=DEV)
    freqs, scale = K.rotary_frequencies(rd, scaling={'kind': 'by_parts', 'factor': 4, 'window': 512}, device=DEV)
    for p in (pos, pos.int()):
        y = K.rotary(x, p, freqs, heads, layout, scale)
        rotary_close(y, rotary_ref(x, pos, freqs, heads, layout, scale), dt)
    back = K.rotary(x, pos, freqs, heads, layout, scale, inverse=True)
    rotary_close(back, rotary_ref(x, pos, freqs, heads, layout, scale, -1.0), dt)
    z = x.clone()
    assert K.rotary(z, pos, freqs, heads, layout, scale, out=z) is z and torch.equal(z, y)   # in place
    # columns of a wider matrix, unaligned: the same bits, nothing else written
    wide = randn(g, rows, heads * hd + 13, dt=dt)
    wide[:, 5:5 + heads * hd] = x
    out = torch.full_like(wide, 7.0)
    K.rotary(wide[:, 5:5 + heads * hd], pos, freqs, heads, layout, scale, out=out[:, 5:5 + heads * hd])
    assert torch.equal(out[:, 5:5 + heads * hd], y) and bool((out[:, :5] == 7).all() and (out[:, -8:] == 7).all())


def test_rotary_far_positions_keep_their_angle(K):
    """Scores depend on the distance alone, also 10^9 positions out: an fp32 angle would be
    off by tens of radians there."""
    freqs, _ = K.rotary_frequencies(64, device=DEV)
    g = gen('far')
    q, k = randn(g, 1, 64).expand(50, 64).contiguous(), randn(g, 1, 64).expand(50, 64).contiguous()
    lag = torch.arange(50, device=DEV)
    near = (K.rotary(q, lag + 10, freqs, 1) * K.rotary(k, torch.full_like(lag, 10), freqs, 1)).sum(1)
    off = 10 ** 9
    far = (K.rotary(q, lag + off, freqs, 1) * K.rotary(k, torch.full_like(lag, off), freqs, 1)).sum(1)
    # each side: 64 products of elements off by 12 * 2^-24 (|a| + |b|); fp64 angles at 10^9: 2 pi 10^9 2^-53
    lim = 4 * 12 * 2.0 ** -24 * float(q[0].abs().sum() * k[0].abs().max()) + 64 * 1e-6
    assert float((near - far).abs().max()) < lim


def test_rotary_gradient(K, G):
    g = gen('rotg')
    x = randn(g, 6, 5, 3 * 24).requires_grad_(True)
    pos = torch.randint(0, 999, (6, 5), generator=g, device=DEV)
    freqs, _ = K.rotary_frequencies(16, device=DEV)
    for layout in ('half', 'interleaved'):
        y = G.rotary(x, pos, freqs, 3, layout, 1.25)
        dy = randn(g, *y.shape)
        dx, = torch.autograd.grad(y, x, dy)
        ref = rotary_ref(dy.view(30, -1), pos.view(-1), freqs, 3, layout, 1.25, -1.0)
        rotary_close(dx.view(30, -1), ref, torch.float32)
        # a linear map: <dy, R v> = <R^T dy, v> for any v
        v = randn(g, *x.shape)
        lhs = (dy.double() * G.rotary(v, pos, freqs, 3, layout, 1.25).double()).sum()
        rhs = (dx.double() * v.double()).sum()
        assert abs(float(lhs - rhs)) <= 2 * 12 * 2.0 ** -24 * 1.25 * 2 * float((dy.abs() * v.abs()).sum()) + 1e-3
    dx, = torch.autograd.grad(G.rotary(x, pos, freqs, 3).sum(), x)   # an expanded gradient
    assert bool(torch.isfinite(dx).all())


def test_rotary_refusals(K):
    from tencent_recommendation_2025_amd._lib import GrkError
    x = torch.zeros(8, 128, device=DEV)
    pos, f = torch.zeros(8, dtype=torch.int64, device=DEV), torch.ones(32, dtype=torch.float64, device=DEV)
    for bad in (lambda: K.rotary(x, pos[:7], f, 2), lambda: K.rotary(x, pos.float(), f, 2),
                lambda: K.rotary(x, pos, f.float(), 2), lambda: K.rotary(x, pos, f, 3),
                lambda: K.rotary(x, pos, f, 4), lambda: K.rotary(x, pos, f, 2, 'pairs'),
                lambda: K.rotary(x.double(), pos, f, 2), lambda: K.rotary(x.t(), pos, f, 2),
                lambda: K.rotary(x[:, :64], pos, f, 1, out=x[:, 32:96]),
                lambda: K.rotary(x[:1].expand(8, 128), pos, f, 2)):
        with pytest.raises(GrkError):
            bad()


# ------------------------------------------------------ decayed attention ----
def decays(H):
    return torch.log1p(-torch.exp2(-torch.linspace(3.0, 8.0, H, device=DEV)))


def decay_ref(q, k, v, lg, valid, scale, do=None, state=None):
    """Straight from o_i = scale sum_{j <= i} g^(i - j) (q_i . k_j) v_j in 64 bits: q, k, v
    [B, T, H, d], valid [B, T]; ([B, T, H, d], final state[, dq, dk, dv])."""
    B, T, H, d = q.shape
    m = valid[..., None, None]
    q, k, v = (torch.where(m, x.double(), 0.0).transpose(1, 2).contiguous() for x in (q, k, v))
    lg = lg.double().clamp(max=0.0)
    t = torch.arange(T, device=DEV)
    lag = (t[:, None] - t[None, :]).clamp(min=0)

    def power(n):   # [H, ...]: g^n, g^0 = 1 also for g = 0
        e = lg.view(-1, *[1] * n.dim()) * n
        return torch.where(n == 0, torch.ones_like(e), torch.exp(e))

    D = power(lag) * (t[:, None] >= t[None, :])
    P = torch.matmul(q, k.transpose(-1, -2).contiguous()) * D
    o = torch.matmul(P, v)
    S = torch.matmul((k * power(T - 1 - t)[..., None]).transpose(-1, -2).contiguous(), v)
    if state is not None:
        s0 = state.double()
        o = o + torch.matmul(q, s0) * power(t + 1)[..., None]
        S = S + s0 * power(torch.tensor(T, device=DEV))[:, None, None]
    back = lambda x: (x.transpose(1, 2) * m).reshape(B * T, H * d)  # noqa: E731
    if do is None:
        return back(scale * o), S
    do = torch.where(m, do.double(), 0.0).transpose(1, 2).contiguous()
    dP = torch.matmul(do, v.transpose(-1, -2).contiguous()) * D
    tr = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    return back(scale * o), S, back(scale * torch.matmul(dP, k)), back(scale * torch.matmul(tr(dP), q)), \
        back(scale * torch.matmul(tr(P), do))


def decay_tol(dt):
    return (3 if dt == torch.bfloat16 else 1) * u_of(dt) + 300 * 2.0 ** -24


def mask_of(kind, B, T, g):
    t = torch.arange(T, device=DEV)
    n = torch.randint(1, T + 1, (B,), generator=g, device=DEV)
    left = t[None, :] >= (T - n)[:, None]
    if kind == 'none':
        return None
    if kind == 'left':
        return left
    if kind == 'holes':
        return left & (torch.rand(B, T, generator=g, device=DEV) > 0.2)
    valid = left & (torch.rand(B, T, generator=g, device=DEV) > 0.2)   # 'empty': a row with nothing, and the last step too
    valid[0] = False
    valid[:, -1] = False
    return valid


SHAPES = [(1, 1, 1, 64), (3, 2, 2, 16), (2, 63, 1, 64), (2, 64, 3, 33), (3, 65, 2, 128), (2, 201, 8, 64), (1, 700, 2, 64),
          (2, 513, 2, 20), (1, 1100, 1, 72), (5, 130, 1, 32), (1, 300, 2, 1), (2, 90, 2, 127)]


@pytest.mark.parametrize('mask', ['none', 'left', 'holes', 'empty'])
@pytest.mark.parametrize('dt', list(DT))
@pytest.mark.parametrize('B,T,H,hd', SHAPES)
def test_decay_attn(K, G, B, T, H, hd, dt, mask):
    dt = DT[dt]
    g = gen('decay', B, T, H, hd, mask)
    D = H * hd
    qkv = randn(g, B * T, 3 * D, dt=dt)
    do = randn(g, B * T, D, dt=dt)
    lg, scale = decays(H), hd ** -0.5
    valid = mask_of(mask, B, T, g)
    kv = None if valid is None else valid.to(torch.uint8)
    if valid is not None:   # what lies in masked rows is never used
        gone = (~valid).view(-1)
        qkv[gone] = torch.tensor([float('nan'), float('inf'), float('-inf'), torch.finfo(dt).min], device=DEV,
                                 dtype=dt)[torch.randint(0, 4, (int(gone.sum()), 3 * D), generator=g, device=DEV)]
        do[gone] = float('nan')
    split = [x.reshape(B, T, H, hd) for x in qkv.split(D, 1)]
    ones = torch.ones(B, T, dtype=torch.bool, device=DEV)
    want = decay_ref(*split, lg, ones if valid is None else valid, scale, do.view(B, T, H, hd))
    x = qkv.clone().requires_grad_(True)
    o = G.decay_attn(x, lg, B, T, key_valid=kv)
    tol = decay_tol(dt)
    close(o.detach(), want[0], tol)
    dx, = torch.autograd.grad(o, x, do)
    for got, ref in zip(dx.split(D, 1), want[2:]):
        close(got, ref, tol)
    if valid is not None:
        assert bool((o[gone] == 0).all() and (dx[gone] == 0).all())
    # separate matrices at odd offsets give what the packed rows give, and the state
    off = [torch.cat([randn(g, B * T, 3, dt=dt), s, randn(g, B * T, 2, dt=dt)], 1)[:, 3:3 + D] for s in qkv.split(D, 1)]
    o2, st = K.decay_attn_fwd(*off, lg, B, T, key_valid=kv, return_state=True)
    close(o2, want[0], tol)
    close(st.reshape(B * H, -1), want[1].reshape(B * H, -1), 300 * 2.0 ** -24)   # fp32 whatever the rows are


@pytest.mark.parametrize('dt', list(DT))
@pytest.mark.parametrize('T,hd', [(45, 64), (33, 40), (1, 56)])
def test_decay_attn_many_sequences(K, T, hd, dt):
    """More (sequence, head) pairs than workgroups that run at once, with states."""
    dt = DT[dt]
    B, H = 300, 7
    g = gen('many', T, hd)
    valid = mask_of('holes', B, T, g)
    q, k, v, do = (randn(g, B * T, H * hd, dt=dt) for _ in range(4))
    s0, lg = randn(g, B, H, hd, hd), decays(H)
    heads = lambda x: x.view(B, T, H, hd)  # noqa: E731
    kv = valid.to(torch.uint8)
    want = decay_ref(heads(q), heads(k), heads(v), lg, valid, hd ** -0.5, state=s0)
    o, s = K.decay_attn_fwd(q, k, v, lg, B, T, key_valid=kv, state=s0, return_state=True)
    close(o, want[0], decay_tol(dt))
    close(s.view(B * H, -1), want[1].view(B * H, -1), 300 * 2.0 ** -24)
    want = decay_ref(heads(q), heads(k), heads(v), lg, valid, hd ** -0.5, heads(do))
    close(K.decay_attn_fwd(q, k, v, lg, B, T, key_valid=kv), want[0], decay_tol(dt))
    for a, b in zip(K.decay_attn_bwd(do, q, k, v, lg, B, T, key_valid=kv), want[2:]):
        close(a, b, decay_tol(dt))


def test_decay_attn_extreme_decays(K):
    """g = 1 (0, and above 0), g = 0 (-inf) and a decay that underflows inside a chunk."""
    lg = torch.tensor([0.0, 3.0, float('-inf'), -50.0], device=DEV)
    g = gen('extreme')
    for dt in DT.values():
        q, k, v = (randn(g, 150, 4 * 32, dt=dt) for _ in range(3))
        do = randn(g, 150, 4 * 32, dt=dt)
        want = decay_ref(*(x.view(1, 150, 4, 32) for x in (q, k, v)), lg, torch.ones(1, 150, dtype=torch.bool, device=DEV),
                         0.5, do.view(1, 150, 4, 32))
        o, s = K.decay_attn_fwd(q, k, v, lg, 1, 150, scale=0.5, return_state=True)
        close(o, want[0], decay_tol(dt))
        close(s.view(4, -1), want[1].view(4, -1), 300 * 2.0 ** -24)
        for a, b in zip(K.decay_attn_bwd(do, q, k, v, lg, 1, 150, scale=0.5), want[2:]):
            close(a, b, decay_tol(dt))


@pytest.mark.parametrize('dt', list(DT))
@pytest.mark.parametrize('cut,T', [(1, 2), (64, 128), (100, 333), (1500, 2200)])
def test_decay_attn_continues_from_a_state(K, cut, T, dt):
    """A sequence read in two calls, the second from the first one's state (in place),
    equals the sequence read at once; and both equal the reference."""
    dt = DT[dt]
    B, H, hd = 2, 2, 64
    g = gen('cont', cut, T)
    q, k, v = (randn(g, B, T, H * hd, dt=dt) for _ in range(3))
    s0 = randn(g, B, H, hd, hd)
    lg = decays(H)
    part = lambda x, a, b: x[:, a:b].reshape(-1, H * hd)  # noqa: E731
    whole, s = K.decay_attn_fwd(*(part(x, 0, T) for x in (q, k, v)), lg, B, T, state=s0, return_state=True)
    want, sw = decay_ref(*(x.view(B, T, H, hd) for x in (q, k, v)), lg, torch.ones(B, T, dtype=torch.bool, device=DEV),
                         hd ** -0.5, state=s0)
    close(whole, want, decay_tol(dt))
    close(s.view(B * H, -1), sw.view(B * H, -1), 300 * 2.0 ** -24)
    st = s0.clone()
    o1 = K.decay_attn_fwd(*(part(x, 0, cut) for x in (q, k, v)), lg, B, cut, state=st, return_state=True, state_out=st)[0]
    o2 = K.decay_attn_fwd(*(part(x, cut, T) for x in (q, k, v)), lg, B, T - cut, state=st, return_state=True,
                          state_out=st)[0]
    both = torch.cat([o1.view(B, cut, -1), o2.view(B, T - cut, -1)], 1).view(B * T, -1)
    close(both, want, decay_tol(dt))
    close(st.view(B * H, -1), sw.view(B * H, -1), 300 * 2.0 ** -24)


def test_decay_attn_empty_calls(K):
    lg = decays(2)
    e = torch.empty(0, 128, device=DEV)
    s0 = randn(gen('e'), 3, 2, 64, 64)
    o, s = K.decay_attn_fwd(e, e, e, lg, 3, 0, state=s0, return_state=True)
    assert o.shape == (0, 128) and torch.equal(s, s0)
    assert K.decay_attn_fwd(e, e, e, lg, 0, 9).shape == (0, 128)
    assert [t.shape for t in K.decay_attn_bwd(e, e, e, e, lg, 3, 0)] == [(0, 128)] * 3
    # sequences whose range starts behind their last position
    x = randn(gen('e2'), 10, 128)
    rng = torch.tensor([[5, 0, 0], [5, 0, 1]], dtype=torch.int32, device=DEV)
    o, s = K.decay_attn_fwd(x, x, x, lg, 2, 5, seq_range=rng, state=s0[:2].contiguous(), return_state=True)
    assert bool((o == 0).all())
    close(s.view(4, -1), (s0[:2].double() * torch.exp(5 * lg.double())[:, None, None]).view(4, -1), 300 * 2.0 ** -24)


@pytest.mark.parametrize('dt', list(DT))
@pytest.mark.parametrize('B,T,H,hd', [(5, 201, 2, 64), (3, 1025, 1, 128), (40, 33, 4, 16)])
def test_decay_attn_packed_rows(K, B, T, H, hd, dt):
    """The packed rows of a left-padded batch (holes inside, one sequence with nothing)
    equal the padded batch; the rows behind the last sequence come out zero."""
    dt = DT[dt]
    g = gen('packed', B, T)
    D = H * hd
    valid = mask_of('holes', B, T, g)
    valid[:, -1] = True
    valid[1] = False
    kv = valid.to(torch.uint8)
    n = int((T - torch.where(valid.any(1), valid.int().argmax(1), T)).sum())
    rng, base, rmap, _ = K.jagged_layout(kv, n + 37)
    x, do = randn(g, B * T, 3 * D, dt=dt), randn(g, B * T, D, dt=dt)
    rows = rmap.long()
    packed = torch.full((n + 37, 3 * D), float('nan'), device=DEV, dtype=dt)
    pdo = torch.full((n + 37, D), float('nan'), device=DEV, dtype=dt)
    packed[:n], pdo[:n] = x[rows[:n]], do[rows[:n]]
    lg = decays(H)
    for kw in (dict(key_valid=kv), dict(key_valid=kv, seq_range=rng)):
        o = K.decay_attn_fwd(*x.split(D, 1), lg, B, T, **kw)
        d = K.decay_attn_bwd(do, *x.split(D, 1), lg, B, T, **kw)
        po = K.decay_attn_fwd(*packed.split(D, 1), lg, B, T, key_valid=kv, seq_range=rng, row_base=base)
        pd = K.decay_attn_bwd(pdo, *packed.split(D, 1), lg, B, T, key_valid=kv, seq_range=rng, row_base=base)
        for full, pk in zip((o, *d), (po, *pd)):
            close(pk[:n], full[rows[:n]], decay_tol(dt))
            assert bool((pk[n:] == 0).all())
    want = decay_ref(*(s.reshape(B, T, H, hd) for s in x.split(D, 1)), lg, valid, hd ** -0.5, do.view(B, T, H, hd))
    for a, b in zip((o, *d), (want[0], *want[2:])):
        close(a, b, decay_tol(dt))


@pytest.mark.parametrize('dt', list(DT))
def test_the_order_of_the_sequences_is_free(K, dt):
    """Ranges list the sequences longest first; any order that names each once gives the
    same bits, packed and padded, in one segment and in several."""
    dt = DT[dt]
    g = gen('order')
    for B, T, H, hd in ((9, 70, 2, 32), (3, 1100, 1, 64)):
        kv = mask_of('left', B, T, g)
        kv[:, -1] = True
        kv = kv.to(torch.uint8)
        n = int(kv.sum())
        rng, base, _, _ = K.jagged_layout(kv, n)
        D = H * hd
        x, do, lg = randn(g, n, 3 * D, dt=dt), randn(g, n, D, dt=dt), decays(H)
        xp, dp = randn(g, B * T, 3 * D, dt=dt), randn(g, B * T, D, dt=dt)
        got = []
        for order in (rng[:, 2], torch.arange(B, device=DEV), torch.randperm(B, generator=g, device=DEV)):
            r = rng.clone()
            r[:, 2] = order
            kw, kp = dict(key_valid=kv, seq_range=r, row_base=base), dict(key_valid=kv, seq_range=r)
            got.append([K.decay_attn_fwd(*x.split(D, 1), lg, B, T, **kw), *K.decay_attn_bwd(do, *x.split(D, 1), lg, B, T, **kw),
                        *K.decay_attn_fwd(*xp.split(D, 1), lg, B, T, return_state=True, **kp),
                        *K.decay_attn_bwd(dp, *xp.split(D, 1), lg, B, T, **kp)])
        for other in got[1:]:
            assert all(torch.equal(a, b) for a, b in zip(got[0], other))


def test_decay_attn_gradient_against_differences(G):
    """o is linear in each of q, k, v: along a direction e its central difference over
    2 h is the derivative plus h^2 times the cubic term o(e_q, e_k, e_v)."""
    g = gen('fd')
    B, T, H, hd, h = 2, 90, 2, 32, 0.25
    D = H * hd
    lg = decays(H)
    x, e = randn(g, B * T, 3 * D).requires_grad_(True), randn(g, B * T, 3 * D)
    do = randn(g, B * T, D)
    kv = (torch.rand(B, T, generator=g, device=DEV) > 0.1).to(torch.uint8)
    f = lambda z: (G.decay_attn(z, lg, B, T, key_valid=kv).double() * do).sum()  # noqa: E731
    dx, = torch.autograd.grad(G.decay_attn(x, lg, B, T, key_valid=kv), x, do)
    with torch.no_grad():
        diff = (f(x + h * e) - f(x - h * e)) / (2 * h) - h * h * f(e)
        parts = float(f(x + h * e).abs() + f(x - h * e).abs()) / (2 * h)
    want = (dx.double() * e).sum()
    # two sums of B T D products, each off by about 300 * 2^-24 of its size
    size = float((do.abs() * G.decay_attn(x.detach(), lg, B, T, key_valid=kv).abs()).sum()) / h + parts + float((dx * e).abs().sum())
    assert abs(float(diff - want)) <= 300 * 2.0 ** -24 * size


# -------------------------------------------------------------- single events --
@pytest.mark.parametrize('dt', list(DT))
@pytest.mark.parametrize('H,hd', [(2, 64), (3, 33), (1, 128), (8, 4), (2, 1), (1, 72)])
def test_decay_step_is_the_sequence(K, H, hd, dt):
    """T single events per user, one call each, equal the sequences read at once."""
    dt = DT[dt]
    n, T = 5, 20
    g = gen('step', H, hd)
    q, k, v = (randn(g, n, T, H * hd, dt=dt) for _ in range(3))
    lg = decays(H)
    s0 = randn(g, n, H, hd, hd)
    want, sw = decay_ref(*(x.view(n, T, H, hd) for x in (q, k, v)), lg, torch.ones(n, T, dtype=torch.bool, device=DEV),
                         0.3, state=s0)
    pool = randn(g, 9, H, hd, hd)
    slots = torch.tensor([7, 0, 3, 8, 2], device=DEV)
    pool[slots] = s0
    rest = pool.clone()
    for t in range(T):
        o = K.decay_attn_step(q[:, t].contiguous(), k[:, t], v[:, t], lg, pool, slots if t % 2 else slots.int(), scale=0.3)
        close(o, want.view(n, T, -1)[:, t], u_of(dt) + 300 * 2.0 ** -24)
    close(pool[slots].view(n * H, -1), sw.view(n * H, -1), 300 * 2.0 ** -24)
    for s in (1, 4, 5, 6):
        assert torch.equal(pool[s], rest[s])
    own = s0.clone()   # without slots: event i, state i
    o = K.decay_attn_step(q[:, 0], k[:, 0], v[:, 0], lg, own, scale=0.3)
    close(o, want.view(n, T, -1)[:, 0], u_of(dt) + 300 * 2.0 ** -24)


@pytest.mark.parametrize('n', [7, 400, 1500])
def test_decay_step_slots_that_repeat_or_hold_nothing(K, n):
    """Events of one slot are taken in their order; a negative slot holds no event, one past
    the states sets the flag; both leave every state as it is."""
    H, hd = 2, 16
    g = gen('slots', n)
    q, k, v = (randn(g, n, H * hd) for _ in range(3))
    lg = decays(H)
    pool = randn(g, 12, H, hd, hd)
    slots = torch.randint(0, 10, (n,), generator=g, device=DEV)
    slots[2], slots[4] = -1, 12
    want_pool, want = pool.double().clone(), torch.zeros(n, H, hd, dtype=torch.float64, device=DEV)
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < 12:
            want_pool[s] = want_pool[s] * torch.exp(lg.double())[:, None, None] \
                + k[i].double().view(H, hd, 1) * v[i].double().view(H, 1, hd)
            want[i] = (q[i].double().view(H, 1, hd) @ want_pool[s])[:, 0]
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    o = K.decay_attn_step(q, k, v, lg, pool, slots, scale=1.0, err_flag=flag)
    close(o, want.view(n, -1), 300 * 2.0 ** -24)
    close(pool.view(12, -1), want_pool.view(12, -1), 300 * 2.0 ** -24)
    assert int(flag) == 1 and bool((o[2] == 0).all() and (o[4] == 0).all())
    slots[4] = 0
    flag.zero_()
    K.decay_attn_step(q, k, v, lg, pool, slots, err_flag=flag)
    assert int(flag) == 0


def test_decay_step_far_in_a_large_pool(K):
    """State offsets past 2^31 elements."""
    H, hd = 8, 64
    slots_n = 2 ** 31 // (H * hd * hd) + 5
    pool = torch.empty(slots_n, H, hd, hd, device=DEV)
    g = gen('large')
    q, k, v = (randn(g, 2, H * hd) for _ in range(3))
    s0 = randn(g, 2, H, hd, hd)
    slots = torch.tensor([slots_n - 1, 1], device=DEV)
    pool[slots] = s0
    lg = decays(H)
    want, sw = decay_ref(*(x.view(2, 1, H, hd) for x in (q, k, v)), lg, torch.ones(2, 1, dtype=torch.bool, device=DEV),
                         hd ** -0.5, state=s0)
    o = K.decay_attn_step(q, k, v, lg, pool, slots)
    close(o, want, 300 * 2.0 ** -24)
    close(pool[slots].view(2 * H, -1), sw.view(2 * H, -1), 300 * 2.0 ** -24)


def test_a_decay_that_is_no_number_shows(K):
    """NaN in log_decay reaches every later event of its head, and no other head."""
    lg = torch.tensor([-0.1, float('nan')], device=DEV)
    g = gen('nan decay')
    for dt in DT.values():
        q, k, v = (randn(g, 300, 2 * 32, dt=dt) for _ in range(3))
        o, s = K.decay_attn_fwd(q, k, v, lg, 1, 300, return_state=True)
        want = K.decay_attn_fwd(q, k, v, torch.full((2,), -0.1, device=DEV), 1, 300, return_state=True)[0]
        assert torch.equal(o[:, :32], want[:, :32]) and bool(o[1:, 32:].isnan().all()) and bool(s[0, 1].isnan().all())
        state = torch.ones(1, 2, 32, 32, device=DEV)
        e = K.decay_attn_step(q[:1], k[:1], v[:1], lg, state)
        assert bool(e[:, 32:].isnan().all()) and not bool(e[:, :32].isnan().any())
        assert bool(state[:, 1].isnan().all()) and not bool(state[:, 0].isnan().any())


def test_results_may_not_lie_on_operands(K):
    from tencent_recommendation_2025_amd._lib import GrkError
    lg = decays(2)
    x = torch.zeros(10, 128, device=DEV)
    pool = torch.zeros(4, 2, 64, 64, device=DEV)
    in_pool = pool.view(-1, 128)[:10]
    for bad in (lambda: K.decay_attn_fwd(x, x, x, lg, 2, 5, state=pool[:2], state_out=pool[1:3]),
                lambda: K.decay_attn_fwd(x, x, in_pool, lg, 2, 5, state_out=pool[:2]),
                lambda: K.decay_attn_fwd(x, x, x, lg, 2, 5, state=pool[:2], out=in_pool),
                lambda: K.decay_attn_fwd(x, x, x, lg, 2, 5, state_out=pool[:2], out=in_pool),
                lambda: K.decay_attn_step(x[:4], x[:4], x[:4], lg, pool, out=in_pool[:4]),
                lambda: K.decay_attn_fwd(x, x, x, lg, 2, 5, out=x[0]),
                lambda: K.rotary(x, torch.zeros(10, dtype=torch.int64, device=DEV),
                                 torch.ones(32, dtype=torch.float64, device=DEV), 2, out=x[1]),
                lambda: K.head_norm_bwd(x[0], x, None, None, 2, dx=torch.empty_like(x))):
        with pytest.raises(GrkError):
            bad()
    # the states in place are fine
    o, s = K.decay_attn_fwd(x, x, x, lg, 2, 5, state=pool[:2], return_state=True, state_out=pool[:2])
    assert s.data_ptr() == pool.data_ptr()


def test_decay_refusals(K):
    from tencent_recommendation_2025_amd._lib import GrkError
    lg = decays(2)
    x = torch.zeros(10, 128, device=DEV)
    ok = dict(batch=2, seq_len=5)
    f = lambda q=x, k=x, v=x, l=lg, **kw: K.decay_attn_fwd(q, k, v, l, **{**ok, **kw})  # noqa: E731
    base = torch.zeros(3, dtype=torch.int64, device=DEV)
    rng = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    for bad in (lambda: f(l=lg.double()), lambda: f(k=x[:, :64]), lambda: f(k=x.bfloat16()), lambda: f(q=x.double()),
                lambda: f(seq_len=6), lambda: f(key_valid=torch.ones(2, 5, device=DEV)),
                lambda: f(key_valid=torch.ones(5, 2, dtype=torch.uint8, device=DEV)), lambda: f(row_base=base),
                lambda: f(seq_range=rng.long()), lambda: f(out=x), lambda: f(state=torch.zeros(2, 2, 64, 32, device=DEV)),
                lambda: f(q=torch.zeros(10, 300, device=DEV), k=torch.zeros(10, 300, device=DEV),
                          v=torch.zeros(10, 300, device=DEV)),
                lambda: f(v=x.t().contiguous().t()), lambda: f(key_valid=torch.ones(2, 5, dtype=torch.uint8)),
                lambda: K.decay_attn_bwd(x, x, x, x, lg, 2, 5, dq=x),
                lambda: K.decay_attn_step(x, x, x, lg, torch.zeros(9, 2, 64, 64, device=DEV)),
                lambda: K.decay_attn_step(x, x, x, lg, torch.zeros(10, 2, 64, 64, device=DEV, dtype=torch.bfloat16)),
                lambda: K.decay_attn_step(x, x, x, lg, torch.zeros(10, 2, 64, 64, device=DEV), slots=rng)):
        with pytest.raises(GrkError):
            bad()


# --------------------------------------------------------------- head norm ----
def norm_ref(x, w, b, heads, eps, gate, dy):
    N, D = x.shape
    leaves = [t.double().requires_grad_(True) if t is not None else None for t in (x, w, b, gate)]
    z = leaves[0].view(N, heads, D // heads)
    c = z - z.mean(-1, keepdim=True)
    f = (c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)).reshape(N, D)
    if w is not None:
        f = f * leaves[1]
    if b is not None:
        f = f + leaves[2]
    if gate is not None:
        f = f * leaves[3] * torch.sigmoid(leaves[3])
    got = torch.autograd.grad(f, [t for t in leaves if t is not None], dy.double())
    it = iter(got)
    return f.detach(), [next(it) if t is not None else None for t in leaves]


@pytest.mark.parametrize('dt', list(DT))
@pytest.mark.parametrize('gated', [False, True])
@pytest.mark.parametrize('rows,heads,hd', [(1, 1, 8), (64, 8, 64), (1001, 8, 64), (300, 3, 24), (37, 16, 128), (513, 1, 1000),
                                           (9, 2, 1024), (33, 1, 2048), (200, 5, 7), (77, 2, 50), (40, 1, 301), (5, 1, 2047),
                                           (700, 300, 8), (3000, 1, 1)])
def test_head_norm(K, G, rows, heads, hd, gated, dt):
    dt = DT[dt]
    g = gen('norm', rows, heads, hd)
    D = heads * hd
    x = (3 * randn(g, rows, D) + 10 * randn(g, rows, 1)).to(dt)
    gate = randn(g, rows, D, dt=dt) if gated else None
    w, b = 1 + 0.3 * randn(g, D), 0.3 * randn(g, D)
    dy = randn(g, rows, D, dt=dt)
    eps = 1e-5
    y = K.head_norm_fwd(x, w, b, heads, eps, gate)
    dx, dg, dw, db = K.head_norm_bwd(dy, x, w, b, heads, eps, gate)
    ry, (rx, rw, rb, rg) = norm_ref(x, w, b, heads, eps, gate, dy)
    tol = u_of(dt) + 320 * 2.0 ** -24
    close(y, ry, tol)
    if hd > 2:   # of one or two columns the gradient is a difference that cancels but for eps
        close(dx, rx, 2 * tol, rows=False)
    if gated:
        close(dg, rg, tol)
    sums = 320 * 2.0 ** -24
    close(dw, rw, sums if hd > 1 else 1e9)
    close(db, rb, sums)
    dx2, dg2, dw2, db2 = K.head_norm_bwd(dy, x, w, b, heads, eps, gate)
    assert torch.equal(dw, dw2) and torch.equal(db, db2) and torch.equal(dx, dx2)   # the same bits every run
    # odd offsets and strides: the same numbers, nothing else written
    wide = torch.zeros(rows, D + 9, device=DEV, dtype=dt)
    wide[:, 3:3 + D] = x
    out = torch.full_like(wide, 7.0)
    K.head_norm_fwd(wide[:, 3:3 + D], w, b, heads, eps, gate, out=out[:, 3:3 + D])
    close(out[:, 3:3 + D], ry, tol)
    assert bool((out[:, :3] == 7).all() and (out[:, -6:] == 7).all())
    # through autograd, without a bias or any affine
    for ww, bb in ((w, None), (None, None)):
        leaf = x.clone().requires_grad_(True)
        got = G.head_norm(leaf, ww, bb, heads, eps, gate)
        r2, (rx2, _, _, _) = norm_ref(x, ww, bb, heads, eps, gate, dy)
        if hd > 1:
            close(got.detach(), r2, tol)
        if hd > 2:
            close(torch.autograd.grad(got, leaf, dy)[0], rx2, 2 * tol, rows=False)


def test_head_norm_of_constant_and_empty_rows(K):
    x = torch.full((5, 64), 3.0, device=DEV)
    x[1] = 0
    w, b = torch.ones(64, device=DEV), torch.full((64,), 0.5, device=DEV)
    assert bool((K.head_norm_fwd(x, w, b, 4) == 0.5).all())
    e = torch.empty(0, 64, device=DEV)
    assert K.head_norm_fwd(e, w, b, 4).shape == (0, 64)
    dx, _, dw, db = K.head_norm_bwd(e, e, w, b, 4)
    assert dx.shape == (0, 64) and bool((dw == 0).all() and (db == 0).all())
    y = K.head_norm_fwd(x, w, b, 4, out=x)   # in place
    assert y is x and bool((x == 0.5).all())


def test_head_norm_under_another_default_dtype(K):
    """The weight gradients' workspace does not follow torch's default dtype."""
    g = gen('default dtype')
    x, dy, w = randn(g, 1000, 256), randn(g, 1000, 256), 1 + 0.2 * randn(g, 256)
    want = K.head_norm_bwd(dy, x, w, w, 4)
    kept = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    try:
        got = K.head_norm_bwd(dy, x, w, w, 4)
    finally:
        torch.set_default_dtype(kept)
    for i in (0, 2, 3):
        assert got[i].dtype == torch.float32 and torch.equal(got[i], want[i])


def test_offsets_past_32_bits(K):
    """Rows whose stride carries them past 2^31 elements."""
    g = gen('far rows')
    ld, n = 2 ** 28 + 8, 11
    buf = torch.empty(ld * n, device=DEV, dtype=torch.bfloat16)
    x = buf.as_strided((n, 128), (ld, 1))
    x.copy_(randn(g, n, 128, dt=torch.bfloat16))
    c = x.contiguous()
    pos, (freqs, _) = torch.arange(n, device=DEV), K.rotary_frequencies(64, device=DEV)
    assert torch.equal(K.rotary(x, pos, freqs, 2), K.rotary(c, pos, freqs, 2))
    assert torch.equal(K.head_norm_fwd(x, None, None, 2), K.head_norm_fwd(c, None, None, 2))
    # attention: strides of 2^24 and more take the general kernel, shorter ones the bf16 kernel
    for ld, n in ((ld, n), (2 ** 23 + 8, 300)):
        buf = torch.empty(ld * n, device=DEV, dtype=torch.bfloat16)
        x = buf.as_strided((n, 128), (ld, 1))
        x.copy_(randn(g, n, 128, dt=torch.bfloat16))
        lg, one = decays(2), x.reshape(1, n, 2, 64)
        want = decay_ref(one, one, one, lg, torch.ones(1, n, dtype=torch.bool, device=DEV), 0.125, one)
        close(K.decay_attn_fwd(x, x, x, lg, 1, n), want[0], decay_tol(torch.bfloat16))
        for a, b in zip(K.decay_attn_bwd(x, x, x, x, lg, 1, n), want[2:]):
            close(a, b, decay_tol(torch.bfloat16))
        out = torch.empty(ld * n, device=DEV, dtype=torch.bfloat16).as_strided((n, 128), (ld, 1))
        close(K.decay_attn_fwd(x, x, x, lg, 1, n, out=out), want[0], decay_tol(torch.bfloat16))


# ------------------------------------------------- graphs, streams, a run of them --
def layer(G, pre, pos, freqs, lg, w, B, T, H, kv):
    """What the decay block does between its two projections."""
    D = pre.shape[1] // 4
    qk = G.rotary(pre[:, 2 * D:], pos, freqs, 2 * H)
    o = G.decay_attn(torch.cat([qk, pre[:, D:2 * D]], 1), lg, B, T, key_valid=kv)
    return G.head_norm(o, w, None, H, 1e-5, gate=pre[:, :D])


def layer_ref(pre, pos, freqs, lg, w, B, T, H, kv, dy):
    D = pre.shape[1] // 4
    hd = D // H
    x = pre.double().requires_grad_(True)
    w = w.double().requires_grad_(True)
    ang = pos.double()[:, None] * freqs
    z = x[:, 2 * D:].view(B * T, 2 * H, 2, hd // 2)
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    qk = torch.stack([z[:, :, 0] * c - z[:, :, 1] * s, z[:, :, 1] * c + z[:, :, 0] * s], 2).reshape(B, T, 2, H, hd)
    m = kv.bool()[..., None, None]
    q, k, v = (torch.where(m, t, 0.0).transpose(1, 2) for t in (qk[:, :, 0], qk[:, :, 1],
                                                                x[:, D:2 * D].reshape(B, T, H, hd)))
    t = torch.arange(T, device=DEV)
    lag = t[:, None] - t[None, :]
    P = (q @ k.transpose(-1, -2)) * torch.exp(lg.double()[:, None, None] * lag.clamp(min=0)) * (lag >= 0)
    o = (hd ** -0.5 * (P @ v)).transpose(1, 2) * m
    cen = o - o.mean(-1, keepdim=True)
    f = (cen / torch.sqrt((cen * cen).mean(-1, keepdim=True) + 1e-5)).reshape(B * T, D) * w
    y = f * x[:, :D] * torch.sigmoid(x[:, :D])
    return (y.detach(), *torch.autograd.grad(y, (x, w), dy.double()))


@pytest.mark.parametrize('dt', list(DT))
def test_the_operators_as_a_layer(K, G, dt):
    """Rotary, attention and norm one after the other, forward and backward, against the
    whole in 64 bits.  Each operator adds its own tolerance; the norm divides by the spread
    of o, so the attention's error passes with a factor of about 1 (2 with its gradient)."""
    dt = DT[dt]
    B, T, H, hd = 3, 150, 4, 32
    g = gen('layer')
    pre = randn(g, B * T, 4 * H * hd, dt=dt)
    kv = mask_of('holes', B, T, g).to(torch.uint8)
    pos = torch.arange(T, device=DEV).repeat(B)
    freqs, _ = K.rotary_frequencies(hd, device=DEV)
    lg, w = decays(H), 1 + 0.2 * randn(g, H * hd)
    dy = randn(g, B * T, H * hd, dt=dt)
    leaf, wl = pre.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = layer(G, leaf, pos, freqs, lg, wl, B, T, H, kv)
    dx, dw = torch.autograd.grad(y, (leaf, wl), dy)
    ry, rx, rw = layer_ref(pre, pos, freqs, lg, w, B, T, H, kv, dy)
    tol = decay_tol(dt) + 3 * u_of(dt) + 320 * 2.0 ** -24
    close(y.detach(), ry, 2 * tol, rows=False)
    close(dx, rx, 6 * tol, rows=False)
    close(dw, rw, 2 * tol)


def test_graph_replays_match_eager(K, G):
    """Two graphs of the layer's forward and backward and of single events, replayed in
    turn with eager work between: every replay has the eager bits on its own inputs."""
    B, T, H, hd = 2, 1200, 2, 64
    D = H * hd
    g = gen('graph')
    freqs, _ = K.rotary_frequencies(hd, device=DEV)
    lg, w = decays(H), 1 + 0.2 * randn(g, D)
    pos = torch.arange(T, device=DEV).repeat(B)
    kv = mask_of('holes', B, T, g).to(torch.uint8)

    def work(x, pool):
        qk = K.rotary(x[:, 2 * D:], pos, freqs, 2 * H)
        q, k, v, u = qk[:, :D], qk[:, D:], x[:, D:2 * D], x[:, :D]
        o, s = K.decay_attn_fwd(q, k, v, lg, B, T, key_valid=kv, return_state=True)
        y = K.head_norm_fwd(o, w, None, H, gate=u)
        do, dg, dw, _ = K.head_norm_bwd(y, o, w, None, H, gate=u)
        d = K.decay_attn_bwd(do, q, k, v, lg, B, T, key_valid=kv)
        e = K.decay_attn_step(q[:300], k[:300], v[:300], lg, pool, slots)
        return y, s, do, dg, dw, *d, e, pool

    slots = torch.randint(0, 40, (300,), generator=g, device=DEV)
    xs = [randn(g, B * T, 4 * D, dt=torch.bfloat16) for _ in range(2)]
    pools = [randn(g, 40, H, hd, hd) for _ in range(2)]
    work(xs[0], pools[0].clone())
    torch.cuda.synchronize()
    graphs, outs, kept = [], [], []
    for x, p in zip(xs, pools):
        sx, sp = x.clone(), p.clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = work(sx, sp)
        graphs.append(gr), outs.append(out), kept.append((sx, sp))
    for turn in range(3):
        for i in (0, 1):
            x = randn(g, B * T, 4 * D, dt=torch.bfloat16)
            kept[i][0].copy_(x)
            kept[i][1].copy_(pools[i])
            graphs[i].replay()
            eager = work(x, pools[i].clone())
            torch.cuda.synchronize()
            for a, b in zip(outs[i], eager):
                assert torch.equal(a, b), (turn, i)


def test_saved_rows_that_come_back_elsewhere(K, G):
    """A gradient whose saved rows were kept on the host, from rows of a wider buffer: they
    come back dense, maybe at their old address."""
    g = gen('saved')
    B, T, H, hd = 2, 70, 2, 32
    wide = randn(g, B * T, 4 * H * hd, dt=torch.bfloat16)
    qkv = wide[:, :3 * H * hd].detach().requires_grad_(True)
    lg, do = decays(H), randn(g, B * T, H * hd, dt=torch.bfloat16)
    want, = torch.autograd.grad(G.decay_attn(qkv, lg, B, T), qkv, do)
    home = {}

    def pack(t):
        home[t.data_ptr()] = t
        return t.data_ptr(), t.cpu().contiguous()

    def unpack(kept):
        at = home[kept[0]]
        if at.shape != (B * T, 3 * H * hd):
            return at
        back = wide.view(-1)[:at.numel()].view(at.shape)   # the old address, another stride
        back.copy_(kept[1])
        return back

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        o = G.decay_attn(qkv, lg, B, T)
    got, = torch.autograd.grad(o, qkv, do)
    assert torch.equal(got, want)


def test_another_stream(K):
    """Two calls at once on two streams do not share a workspace."""
    g = gen('streams')
    lg = decays(1)
    xs = [randn(g, 4000, 64, dt=torch.bfloat16) for _ in range(2)]
    want = [K.decay_attn_fwd(x, x, x, lg, 1, 4000) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = K.decay_attn_fwd(xs[i], xs[i], xs[i], lg, 1, 4000)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
