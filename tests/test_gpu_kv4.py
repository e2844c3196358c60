"""The 4-bit KV cache on the GPU against its definition in 64 bits (``oracle/kv4.py``).

Tolerances of attention.  With A = max_j scale * sum_d |q_d k_jd| a score computed in f32 is off by at
most (d + 8) 2^-24 A, so a probability by twice that relative to itself, and sums over n rows add at
most n 2^-24 more: out by (2 (d + 8) A + n) 2^-24 sum_j p_j |v_j| <= (...) max |v|, a row's weight by
(...) times what it received, plus half a step of the sum.
"""
import math

import numpy as np
import pytest

from oracle import kv4 as ok

pytestmark = pytest.mark.gpu


def _cuda(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _i32(a):
    return _cuda(np.asarray(a, np.int32))


def _rows(rng, shape, spread=1.0):
    strong = np.where(rng.random(shape[-1]) < 0.06, 4.0, 1.0)
    return (rng.standard_normal(shape) * strong * spread).astype(np.float32)


def _filled(ctx, rng, B, nkv, cap, d, track=True):
    """A cache with every slot filled from quantised random rows, and its rows' values."""
    from voxcpm_rs_b200.kv4 import Kv4Cache
    import torch
    c = Kv4Cache(ctx, B, nkv, cap, d, track=track)
    vals = []
    for codes, scales, spread in ((c.k_codes, c.k_scales, 1.0), (c.v_codes, c.v_scales, 0.5)):
        cb, sb = ok.quantise(_rows(rng, (B, nkv, c.capacity, d), spread))
        codes.copy_(torch.from_numpy(cb))
        scales.view(torch.uint8).copy_(torch.from_numpy(sb))
        vals.append(ok.values(cb, sb))
    return c, vals[0], vals[1]


def _raw(c):
    import torch
    return [t.view(torch.uint8).cpu().numpy().copy() for t in (c.k_codes, c.k_scales, c.v_codes, c.v_scales)]


# ------------------------------------------------------------------------------ append, read

def _special_rows(d):
    """Rows where the quantiser can go wrong: zeros, tiny, saturating and infinite values, NaN, ties."""
    g = []
    g.append(np.zeros(16))
    g.append(np.full(16, -0.0))
    g.append(np.linspace(-1, 1, 16) * 1e-5)                                   # no scale: all 0
    g.append(np.array([6 * 2.0 ** -9] + [2.0 ** -9 * t for t in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5)] * 2 + [0]))
    edges = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    g.append(np.concatenate([[6.0], edges, -edges, [0.0]]))                   # scale 1, every tie
    up = np.nextafter(edges.astype(np.float32), np.float32(9))
    dn = np.nextafter(edges.astype(np.float32), np.float32(0))
    g.append(np.concatenate([[6.0], up, -dn, [1.0]]))                         # one step off every tie
    g.append(np.concatenate([[6.0 * 1.125], edges * 1.125, -edges * 1.125, [0.0]]))
    g.append(np.linspace(-3000, 3000, 16))                                    # beyond 6 * 448
    g.append(np.array([6 * m for m in (1.0625,)] + [0.5] * 15))               # amax / 6 on a scale's tie
    g.append(np.array([np.inf] + [1.0] * 15))
    g.append(np.array([1.0, np.nan] + [0.0] * 14))
    g.append(np.array([-np.inf, np.nan] + [1e30] * 14))
    g.append(np.array([1e-45] * 16))
    while len(g) % (d // 16):
        g.append(np.arange(16.0) - 8)
    return np.stack(g).reshape(-1, d).astype(np.float32)


@pytest.mark.parametrize("d", [64, 128])
def test_append_special_values(ctx, d):
    """Codes and scales are the definition's, bit for bit, ties and non-finite values included."""
    from voxcpm_rs_b200.kv4 import Kv4Cache
    import torch
    x = _special_rows(d)
    S = len(x)
    c = Kv4Cache(ctx, 1, 1, S, d)
    k = _cuda(x.reshape(1, S, 1, d))
    v = _cuda(-x.reshape(1, S, 1, d))
    c.append(k, v, _i32([0]))
    for got_c, got_s, src in ((c.k_codes, c.k_scales, x), (c.v_codes, c.v_scales, -x)):
        wc, ws = ok.quantise(src)
        gs = got_s.view(torch.uint8).cpu().numpy()[0, 0, :S]
        assert np.array_equal(gs, ws)
        real = np.repeat(ws != 127, 8, -1)  # codes under a NaN scale stand for NaN whatever they are
        assert np.array_equal(got_c.cpu().numpy()[0, 0, :S][real], wc[real])
    k2, v2 = c.read(S)
    want = ok.values(*ok.quantise(x))
    assert np.array_equal(k2.cpu().numpy()[0, 0], want.astype(np.float32), equal_nan=True)
    assert np.array_equal(v2.cpu().numpy()[0, 0], ok.values(*ok.quantise(-x)).astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("B,S,nkv,d", [(1, 1, 2, 128), (8, 1, 2, 128), (3, 5, 1, 64), (2, 131, 4, 128), (5, 33, 3, 64)])
def test_append_and_read(ctx, B, S, nkv, d):
    """Ragged rows out of a fused projection, at given slots; rows around them stay as they were."""
    import torch
    rng = np.random.default_rng(B * 1000 + S)
    c, _, _ = _filled(ctx, rng, B, nkv, S + 70, d)
    before = _raw(c)
    c.weights.fill_(3.0)
    c.positions.fill_(-7)
    wide = _cuda(_rows(rng, (B, S, (2 * nkv + 3) * d)))
    k = wide[..., 3 * d:(3 + nkv) * d].unflatten(-1, (nkv, d))
    v = wide[..., (3 + nkv) * d:].unflatten(-1, (nkv, d))
    start = rng.integers(0, c.capacity - S + 1, B)
    counts = rng.integers(0, S + 1, B)
    counts[-1] = S
    first = rng.integers(0, 10000, B)
    c.append(k, v, _i32(start), _i32(counts), _i32(first))
    kr, vr = c.read(S, _i32(start), _i32(counts))
    after = _raw(c)
    w, pos = c.weights.cpu().numpy(), c.positions.cpu().numpy()
    for i, x in ((0, k), (2, v)):
        wc, ws = ok.quantise(x.cpu().numpy())
        want_c, want_s = before[i].copy(), before[i + 1].copy()
        for b in range(B):
            n, at = counts[b], start[b]
            want_c[b, :, at:at + n] = wc[b, :n].swapaxes(0, 1)
            want_s[b, :, at:at + n] = ws[b, :n].swapaxes(0, 1)
        assert np.array_equal(after[i], want_c) and np.array_equal(after[i + 1], want_s)
    for b in range(B):
        n, at = counts[b], start[b]
        mine = np.zeros(c.capacity, bool)
        mine[at:at + n] = True
        assert np.all(w[b][:, mine] == 0) and np.all(w[b][:, ~mine] == 3)
        assert np.all(pos[b][:, mine] == first[b] + np.arange(n)) and np.all(pos[b][:, ~mine] == -7)
        for got, i in ((kr, 0), (vr, 2)):
            g = got.cpu().numpy()[b]
            assert np.array_equal(g[:, :n], ok.values(after[i][b, :, at:at + n], after[i + 1][b, :, at:at + n]).astype(np.float32))
            assert np.all(g[:, n:] == 0)
    # without counts and positions: all S tokens, positions are the slots
    c.append(k, v, _i32(start))
    assert np.array_equal(c.positions.cpu().numpy()[0, 0, start[0]:start[0] + S], start[0] + np.arange(S))


# ------------------------------------------------------------------------------------ attend

def _check_attend(ctx, rng, B, nkv, nrep, d, max_len, lens, track, cap=None, garbage=True):
    import torch
    c, k, v = _filled(ctx, rng, B, nkv, cap or max(max_len, 1), d)
    lens = np.asarray(lens)
    if garbage:  # what lies behind a sequence's rows must not matter: NaN scales
        for b in range(B):
            c.k_scales.view(torch.uint8)[b, :, lens[b]:] = 0x7f
            c.v_scales.view(torch.uint8)[b, :, lens[b]:] = 0x7f
    nh = nkv * nrep
    wide = rng.standard_normal((B, (nh + 3) * d)).astype(np.float32)
    q = _cuda(wide)[:, 2 * d:(nh + 2) * d]  # rows of a fused projection
    w0 = rng.random((B, nkv, c.capacity)).astype(np.float32)
    c.weights.copy_(torch.from_numpy(w0))
    out = c.attend(q, _i32(lens), max_len, track=track).cpu().numpy().reshape(B, nh, d)
    qn = wide[:, 2 * d:(nh + 2) * d].reshape(B, nh, d)
    want, got_p = ok.attend(qn, k, v, lens, nrep, 1 / math.sqrt(d))
    n = max(1, int(lens.max(initial=0)))
    kk = np.abs(k[:, :, :n])
    A = max(float((np.abs(qn[b, h]) @ kk[b, h // nrep].T).max()) for b in range(B) for h in range(nh)) / math.sqrt(d)
    rel = (2 * (d + 8) * A + n) * 2.0 ** -24
    assert np.all(np.isfinite(out))
    assert np.abs(out - want).max() <= rel * np.abs(v).max()
    assert np.all(out[lens == 0] == 0)
    w = c.weights.cpu().numpy().astype(np.float64)
    if track:
        there = np.arange(c.capacity)[None, None] < lens[:, None, None]
        full = np.zeros(w.shape)
        full[:, :, :got_p.shape[2]] = got_p
        assert np.all(np.abs(w - (w0 + full)) <= rel * full + 2.0 ** -24 * (w0 + full) * 2)
        assert np.array_equal(w[~np.broadcast_to(there, w.shape)], w0[~np.broadcast_to(there, w.shape)])
    else:
        assert np.array_equal(w, w0)
    # a second call gives the same bits
    again = c.attend(q, _i32(lens), max_len).cpu().numpy().reshape(B, nh, d)
    assert np.array_equal(out, again)


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 127, 129, 300])
def test_attend_lengths(ctx, n, d, track):
    _check_attend(ctx, np.random.default_rng(n * d), 1, 2, 8, d, n, [n], track)


@pytest.mark.parametrize("nkv,nrep", [(1, 1), (2, 3), (3, 7), (1, 8), (2, 9), (1, 16), (1, 20)])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_heads(ctx, nkv, nrep, d):
    _check_attend(ctx, np.random.default_rng(nkv * 100 + nrep), 2, nkv, nrep, d, 203, [203, 77], True)


@pytest.mark.parametrize("d,lens,max_len,cap", [
    (128, [0, 1, 500, 999, 1000], 1000, 1024), (64, [0, 0, 0], 64, 64), (128, [0], 0, 32),
    (128, [4097, 5, 0, 2048, 4096, 4095, 33, 1], 4100, 4128), (64, [9000, 17, 8999], 9001, 9024),
    (128, [3, 40, 7], 2048, 2048)])
def test_attend_ragged(ctx, d, lens, max_len, cap):
    """Sequences of other lengths in one call, empty ones among them, many splits and few."""
    _check_attend(ctx, np.random.default_rng(len(lens)), len(lens), 2, 8, d, max_len, lens, True, cap)


@pytest.mark.parametrize("B,max_len", [(32, 1000), (60, 1400), (37, 515)])
@pytest.mark.parametrize("track", [False, True])
def test_attend_many_sequences(ctx, B, max_len, track):
    """Blocks of all sequences on the GPU at once: fewer tiles in flight where they track."""
    rng = np.random.default_rng(B)
    lens = rng.integers(0, max_len + 1, B)
    lens[:3] = max_len, 0, 1
    _check_attend(ctx, rng, B, 2, 8, 128, max_len, lens, track)


def test_attend_large_scores(ctx):
    """Scores of hundreds, the largest at the end: the running maximum grows in every tile, and
    rows far below it vanish."""
    import torch
    rng = np.random.default_rng(5)
    d, n = 128, 700
    c, k, v = _filled(ctx, rng, 1, 1, n, d)
    ramp = np.linspace(0.1, 40, n)[:, None] * np.ones(d)
    cb, sb = ok.quantise((ramp * np.sign(rng.standard_normal(d))).astype(np.float32)[None, None])
    c.k_codes[:, :, :n] = _cuda(cb)
    c.k_scales.view(torch.uint8)[:, :, :n] = _cuda(sb)
    k = ok.values(cb, sb)
    q = np.sign(k[0, 0, -1]) * rng.uniform(0.2, 2.0, d)
    q = np.stack([q, -q, q * 1e-3, q * 0]).astype(np.float32)
    out = c.attend(_cuda(q.reshape(1, -1)), _i32([n])).cpu().numpy().reshape(4, d)
    want, _ = ok.attend(q[None], k, v, [n], 4, 1 / math.sqrt(d))
    for h in range(4):
        A = float((np.abs(q[h]) @ np.abs(k[0, 0]).T).max()) / math.sqrt(d)
        assert np.abs(out[h] - want[0, h]).max() <= (2 * (d + 8) * A + n) * 2.0 ** -24 * np.abs(v).max()


@pytest.mark.parametrize("qs", [1e-30, 1e-6, 1.0, 3e4])
def test_attend_query_range(ctx, qs):
    """Queries of any magnitude: the scale argument brings the scores back."""
    rng = np.random.default_rng(6)
    d, n = 64, 150
    c, k, v = _filled(ctx, rng, 1, 2, n, d)
    q = (rng.standard_normal((1, 8, d)) * qs).astype(np.float32)
    s = 0.125 / qs
    out = c.attend(_cuda(q.reshape(1, -1)), _i32([n]), scale=s).cpu().numpy().reshape(1, 8, d)
    want, _ = ok.attend(q, k[:, :, :n], v[:, :, :n], [n], 4, np.float32(s))
    A = 0.125 * max(float((np.abs(q[0, h]) @ np.abs(k[0, h // 4, :n]).T).max()) for h in range(8)) / qs
    assert np.abs(out - want).max() <= (2 * (d + 8) * A + n) * 2.0 ** -24 * np.abs(v).max()


def test_attend_nan_row_within(ctx):
    """A NaN row that belongs to the sequence shows in its KV head's outputs and nowhere else."""
    import torch
    rng = np.random.default_rng(7)
    c, _, _ = _filled(ctx, rng, 2, 2, 100, 128)
    q = _cuda(rng.standard_normal((2, 16 * 128)).astype(np.float32))
    ref = c.attend(q, _i32([90, 90]))
    c.k_scales.view(torch.uint8)[1, 0, 40, 3] = 0x7f
    got = c.attend(q, _i32([90, 90]))
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1, 8 * 128:], ref[1, 8 * 128:])
    assert torch.isnan(got[1, :8 * 128]).all()


# ------------------------------------------------------------------------------------- evict

def _check_evict(ctx, rng, B, nkv, d, cap, lens, keep, sink, recent, max_len=None, weights=None, inplace=False, gap=0):
    import torch
    c, _, _ = _filled(ctx, rng, B, nkv, cap, d)
    cap = c.capacity
    w = (rng.random((B, nkv, cap)) ** 4 * 9).astype(np.float32) if weights is None else weights
    pos = np.broadcast_to(np.arange(cap) + gap, (B, nkv, cap)).astype(np.int64).copy()
    for b in range(B):  # an earlier eviction has changed the order
        for h in range(nkv):
            pos[b, h, :lens[b]] = rng.permutation(pos[b, h, :lens[b]])
    seen = np.asarray(lens, np.int32) + gap
    c.weights.copy_(torch.from_numpy(w))
    c.positions.copy_(torch.from_numpy(pos))
    before = _raw(c)
    wo = None if inplace else torch.full_like(c.weights, -5.0)
    po = None if inplace else torch.full_like(c.positions, -5)
    got = c.evict(_i32(lens), _i32(seen), keep, sink, recent, max_len, wo, po).cpu().numpy()
    assert got.tolist() == [min(n, keep) for n in lens]
    after = _raw(c)
    wn = (c.weights if inplace else wo).cpu().numpy()
    pn = (c.positions if inplace else po).cpu().numpy()
    for b in range(B):
        for h in range(nkv):
            src = ok.evict(w[b, h], pos[b, h], lens[b], seen[b], keep, sink, recent)
            m = len(src)
            for x, y in zip(before, after):
                assert np.array_equal(y[b, h, :m], x[b, h, src])
                assert np.array_equal(y[b, h, m:], x[b, h, m:])
            assert np.array_equal(wn[b, h, :m], w[b, h, src], equal_nan=True)
            assert np.array_equal(pn[b, h, :m], pos[b, h, src])
            assert np.array_equal(wn[b, h, m:], w[b, h, m:] if inplace else np.full(cap - m, -5.0, np.float32), equal_nan=True)
            assert np.array_equal(pn[b, h, m:], pos[b, h, m:] if inplace else np.full(cap - m, -5, np.int64))
    if not inplace:
        assert np.array_equal(c.weights.cpu().numpy(), w, equal_nan=True)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("d,n,keep,sink,recent", [
    (128, 1, 1, 0, 0), (128, 2, 1, 0, 0), (128, 2, 1, 1, 0), (64, 33, 32, 4, 8), (128, 100, 99, 0, 0),
    (128, 1000, 17, 4, 13), (64, 1025, 1024, 4, 64), (128, 2000, 1000, 0, 1000), (128, 500, 0, 0, 0),
    (64, 5000, 700, 4, 128), (128, 9001, 4096, 4, 256)])
def test_evict(ctx, d, n, keep, sink, recent, inplace):
    rng = np.random.default_rng(n + keep)
    _check_evict(ctx, rng, 2, 2, d, n + 5, [n, max(0, n - 3)], keep, sink, recent, inplace=inplace, gap=50)


def test_evict_ragged(ctx):
    """Sequences at, below and above the budget, an empty one among them, in one call."""
    _check_evict(ctx, np.random.default_rng(1), 6, 2, 128, 9000, [0, 1, 600, 601, 8999, 4000], 600, 4, 100, max_len=8999)


@pytest.mark.parametrize("B,n", [(1, 1025), (1, 2049), (1, 4097), (1, 10241), (1, 16385), (36, 4100), (40, 2500), (75, 2049)])
def test_evict_shapes(ctx, B, n):
    """Either side of where more blocks share a sequence, for few sequences and for many."""
    rng = np.random.default_rng(n)
    lens = np.concatenate([[n], rng.integers(0, n + 1, B - 1)])
    _check_evict(ctx, rng, B, 2, 64, -(-n // 32) * 32, lens, n // 2 + 1, 4, 100)


def test_evict_long(ctx):
    _check_evict(ctx, np.random.default_rng(2), 1, 1, 64, 131072, [131072], 20000, 4, 1000)


@pytest.mark.parametrize("kind", ["equal", "zero", "two", "signs", "special"])
def test_evict_ties(ctx, kind):
    """Equal weights: the lowest slots stay; -0 is 0, NaN the largest."""
    rng = np.random.default_rng(3)
    B, nkv, cap = 1, 2, 6016
    w = {"equal": np.full((B, nkv, cap), 1.25), "zero": np.zeros((B, nkv, cap)) * np.where(rng.random((B, nkv, cap)) < .5, 1, -1),
         "two": rng.integers(0, 2, (B, nkv, cap)).astype(float), "signs": rng.integers(-2, 3, (B, nkv, cap)) * 0.5,
         "special": rng.choice([np.nan, np.inf, -np.inf, 0.0, 1e-42, 3e38], (B, nkv, cap))}[kind].astype(np.float32)
    for keep in (1, 1500, 3007):
        _check_evict(ctx, rng, B, nkv, 64, cap, [6001], keep, 0, 1, weights=w)


# ---------------------------------------------------------------------- refusals on the device

def test_lengths_out_of_range_are_reported(ctx):
    """A length outside its range: the sequence stays as it was, its output is NaN, the others are
    served, and the next synchronize says so."""
    import torch
    from voxcpm_rs_b200._lib import VX_ERR_ARG, VxError
    rng = np.random.default_rng(8)
    c, k, v = _filled(ctx, rng, 3, 2, 64, 64)
    c.positions.copy_(torch.arange(64).expand(3, 2, 64))
    q = _cuda(rng.standard_normal((3, 4 * 64)).astype(np.float32))

    def reported():
        torch.cuda.synchronize()
        with pytest.raises(VxError) as e:
            ctx.synchronize()
        assert e.value.code == VX_ERR_ARG
        ctx.synchronize()  # told once

    for bad in (-1, 65, 2 ** 31 - 1, -2 ** 31):
        ref = c.attend(q, _i32([64, 10, 64]), 64)  # the other sequences' rows change below
        ctx.synchronize()
        got = c.attend(q, _i32([64, bad, 64]), 64, track=True)
        assert torch.isnan(got[1]).all() and torch.equal(got[0], ref[0]) and torch.equal(got[2], ref[2])
        assert (c.weights[1] == 0).all()
        reported()
        x = _cuda(_rows(rng, (3, 1, 2, 64)))
        before = _raw(c)
        c.append(x, x, _i32([0, bad if bad != 65 else 64, 5]))
        assert all(np.array_equal(p[1], q_[1]) for p, q_ in zip(before, _raw(c)))
        reported()
        c.append(x, x, _i32([0, 0, 5]), _i32([1, bad, 1]))
        assert all(np.array_equal(p[1], q_[1]) for p, q_ in zip(before, _raw(c)))
        reported()
        kr, _ = c.read(8, _i32([0, bad, 0]))
        assert (kr[1] == 0).all()
        reported()
        lens = c.evict(_i32([64, bad, 64]), _i32([64, 64, 64]), 32)
        assert lens.tolist() == [32, bad, 32]
        assert all(np.array_equal(p[1], q_[1]) for p, q_ in zip(before, _raw(c)))
        reported()


def test_arguments_are_refused(ctx):
    """Calls of the C ABI that its checks turn down: nothing is launched, the cache stays as it was."""
    import ctypes as C
    import torch
    from voxcpm_rs_b200 import _lib
    rng = np.random.default_rng(12)
    c, _, _ = _filled(ctx, rng, 2, 2, 9632, 64)
    L, before = _lib.lib(), _raw(c)
    one, n = _i32([1, 1]), torch.zeros(2, device="cuda", dtype=torch.int32)
    x, f = torch.zeros(1 << 16, device="cuda"), torch.zeros(2, 2, 9632, device="cuda")
    p = lambda t, off=0: t.data_ptr() + off  # noqa: E731

    def cache(**kw):
        d = _lib.Kv4C()
        C.memmove(C.addressof(d), c._ref, C.sizeof(d))
        for name, v in kw.items():
            setattr(d, name, v)
        return d

    def append(d, k=x, off=0, bs=128, ts=128, S=1, start=one):
        return L.vx_kv4_append(ctx.h, C.addressof(d), p(k, off), p(x), bs, ts, S, start if start is None else p(start), None,
                               None, None)

    def attend(d, q_off=0, ldq=512, nh=8, lens=one, max_len=32, track=0, ldo=512, ws=None, ws_bytes=0):
        return L.vx_kv4_attend(ctx.h, C.addressof(d), p(x, q_off), ldq, nh, p(lens), max_len, 1.0, track, p(x), ldo, ws,
                               ws_bytes, None)

    def evict(d, lens=one, seen=one, max_len=32, keep=8, sink=0, recent=0, out=n):
        return L.vx_kv4_evict(ctx.h, C.addressof(d), p(lens), p(seen), max_len, keep, sink, recent, p(f), p(f), p(out), None)

    good = cache()
    A, S = _lib.VX_ERR_ARG, _lib.VX_ERR_SHAPE
    bad = [(cache(head_dim=96), S), (cache(capacity=33), S), (cache(capacity=0), S), (cache(capacity=2 ** 30 + 32), S),
           (cache(batch=0), S), (cache(n_kv_heads=0), S), (cache(n_kv_heads=32768), S), (cache(batch=40000), S),
           (cache(k_codes=None), A), (cache(v_scales=c.v_scales.data_ptr() + 8), A)]
    for d, code in bad:
        assert [append(d), attend(d), evict(d)] == [code] * 3
        assert L.vx_kv4_read(ctx.h, C.addressof(d), 1, None, None, p(x), p(x), None) == code
    need = L.vx_kv4_attend_workspace(C.addressof(good), 8, 9632, 1)
    ws = torch.empty(need, device="cuda", dtype=torch.uint8)
    calls = [(append(good, off=4), A), (append(good, bs=130), A), (append(good, ts=2), A), (append(good, S=9633), S),
             (append(good, S=-1), S), (append(good, start=None), A),
             (L.vx_kv4_read(ctx.h, C.addressof(good), 9633, None, None, p(x), p(x), None), S),
             (L.vx_kv4_read(ctx.h, C.addressof(good), -1, None, None, p(x), p(x), None), S),
             (L.vx_kv4_read(ctx.h, C.addressof(good), 1, None, None, p(x, 8), p(x), None), A),
             (attend(good, q_off=8), A), (attend(good, ldq=513), A), (attend(good, ldo=508), A), (attend(good, nh=0), S),
             (attend(good, nh=3), S), (attend(good, nh=130), S), (attend(good, max_len=-1), S),
             (attend(good, max_len=9633), S), (attend(cache(weights=None), track=1), A),
             (attend(good, max_len=9632, track=1), A), (attend(good, max_len=9632, track=1, ws=p(ws), ws_bytes=need - 1), A),
             (attend(good, max_len=9632, track=1, ws=p(ws, 8), ws_bytes=need), A),
             (evict(cache(weights=None)), A), (evict(cache(positions=None)), A), (evict(good, lens=n), A),
             (evict(good, seen=n), A), (evict(good, max_len=9633), S), (evict(good, max_len=-1), S),
             (evict(good, keep=-1), S), (evict(good, sink=4, recent=5), S), (evict(good, sink=-1), S),
             (evict(good, sink=2 ** 31 - 1, recent=2 ** 31 - 1), S)]
    assert [got for got, _ in calls] == [code for _, code in calls]
    torch.cuda.synchronize()
    ctx.synchronize()
    assert all(np.array_equal(a, b) for a, b in zip(before, _raw(c))) and (f == 0).all() and (n == 0).all()
