"""Token sampling on the GPU against its definition in 64 bits (``oracle/sampling.py``): ids are
equal, log-probabilities within one rounding to f32 (2^-24 of the value, and as much of 1 for the
logarithm's argument)."""
import numpy as np
import pytest

from oracle import sampling as osm

pytestmark = pytest.mark.gpu


def _cuda(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _check(ctx, x, u, T=None, k=None, p=None, mp=None, logits=None):
    from voxcpm_rs_b200.sampling import sample
    R = len(x)
    f = lambda a, dt: None if a is None else np.broadcast_to(np.asarray(a, dt), (R,)).copy()  # noqa: E731
    T, k, p, mp, u = f(T, np.float32), f(k, np.int32), f(p, np.float32), f(mp, np.float32), f(u, np.float32)
    c = lambda a: None if a is None else _cuda(a)  # noqa: E731
    ids, lp = sample(ctx, _cuda(x) if logits is None else logits, c(u), c(T), c(k), c(p), c(mp), return_logprob=True)
    ids, lp = ids.cpu().numpy(), lp.cpu().numpy()
    for r in range(R):
        i, l = osm.sample_row(x[r], u[r], 1.0 if T is None else T[r], 0 if k is None else int(k[r]),
                              1.0 if p is None else p[r], 0.0 if mp is None else mp[r])
        assert ids[r] == i, (r, ids[r], i)
        assert (np.isnan(l) and np.isnan(lp[r])) or lp[r] == l or abs(lp[r] - l) <= 2.0 ** -24 * (1 + abs(l)), (r, lp[r], l)
    return ids


def _logits(rng, R, V):
    x = rng.standard_normal((R, V)) * 2.5
    x[rng.random((R, V)) < 0.02] = -np.inf
    x[:, rng.integers(0, V)] += 6
    return x.astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 31, 32, 33, 1000, 4097, 20011])
@pytest.mark.parametrize("mix", ["plain", "topk", "topp", "minp", "all"])
def test_sample(ctx, V, mix):
    rng = np.random.default_rng(V)
    R = 12
    on = lambda m, a: a if mix in (m, "all") else None  # noqa: E731
    _check(ctx, _logits(rng, R, V), rng.random(R), rng.uniform(0.3, 2.0, R), on("topk", rng.integers(-1, 60, R)),
           on("topp", rng.uniform(0.05, 1.05, R)), on("minp", rng.uniform(0.0, 0.5, R)))


@pytest.mark.parametrize("R,V", [(1, 73448), (64, 73448), (200, 5003), (3, 262144), (150, 40000)])
def test_sample_sizes(ctx, R, V):
    rng = np.random.default_rng(R)
    x = _logits(rng, R, V)
    T = np.where(rng.random(R) < 0.2, 0.0, rng.uniform(0.5, 1.2, R))
    some = slice(0, min(R, 6))  # the rows that the definition walks
    from voxcpm_rs_b200.sampling import sample
    u, k, p, mp = rng.random(R), rng.integers(0, 100, R), rng.uniform(0.7, 1.0, R), rng.uniform(0, 0.1, R)
    a = [_cuda(t.astype(dt)) for t, dt in ((u, "f4"), (T, "f4"), (k, "i4"), (p, "f4"), (mp, "f4"))]
    whole = sample(ctx, _cuda(x), *a).cpu().numpy()
    assert whole[some].tolist() == _check(ctx, x[some], u[some], T[some], k[some], p[some], mp[some]).tolist()
    assert np.all((whole >= 0) & (whole < V))


def test_sample_edges(ctx):
    """Rows whose mask leaves nothing, NaN, infinities, ties, the ends of u, settings at their ends."""
    rng = np.random.default_rng(1)
    V = 5000
    ninf = np.full(V, -np.inf, np.float32)
    base = rng.standard_normal(V).astype(np.float32)
    one = ninf.copy()
    one[4321] = -3e38
    nan = base.copy()
    nan[17] = np.nan
    pinf = base.copy()
    pinf[[5, 4000]] = np.inf
    flat = np.zeros(V, np.float32)
    signs = np.where(rng.random(V) < 0.5, 0.0, -0.0).astype(np.float32)
    huge = np.where(rng.random(V) < 0.5, 3e38, -3e38).astype(np.float32)
    rows = np.stack([ninf, one, nan, pinf, flat, signs, huge, base])
    for u in (0.0, 0.5, 1 - 2.0 ** -24, 2.0 ** -30):
        for kw in ({}, dict(k=1), dict(k=7), dict(k=V), dict(k=V + 5), dict(k=-3), dict(p=0.0), dict(p=-1.0), dict(p=0.3),
                   dict(p=1.0), dict(p=1 - 2.0 ** -24), dict(mp=1.0), dict(mp=2.0), dict(mp=0.5), dict(k=9, p=0.5, mp=0.9)):
            _check(ctx, rows, u, **kw)
    for T in (0.0, 1e-30, 1e30, np.inf, -1.0, np.nan):
        _check(ctx, rows, 0.37, T=T)
    # the same index twice: equal logits all over, the prefix goes by the lowest index
    two = rng.integers(0, 3, (4, V)).astype(np.float32)
    for k in (1, 100, 1700, 3400):
        _check(ctx, two, [0.1, 0.5, 0.9, 0.999], k=k, p=0.6)


def test_sample_strided_rows(ctx):
    import torch
    rng = np.random.default_rng(2)
    x = _logits(rng, 5, 777)
    wide = torch.full((5, 1000), float("nan"), device="cuda")
    wide[:, 3:780] = _cuda(x)
    _check(ctx, x, rng.random(5), T=0.8, k=40, logits=wide[:, 3:780])


def test_sample_follows_the_distribution(ctx):
    """u = (i + 1/2) / n walks the distribution: each token comes n * p times, to within one."""
    rng = np.random.default_rng(3)
    V, n = 50, 4000
    x = (rng.standard_normal(V) * 2).astype(np.float32)
    from voxcpm_rs_b200.sampling import sample
    ids = sample(ctx, _cuda(np.broadcast_to(x, (n, V))), _cuda(((np.arange(n) + 0.5) / n).astype(np.float32))).cpu().numpy()
    p = np.exp(x - x.max().astype(np.float64))
    p /= p.sum()
    assert np.abs(np.bincount(ids, minlength=V) - n * p).max() <= 1.5
    assert np.all(np.diff(ids) >= 0)


@pytest.mark.parametrize("kw", [{}, dict(k=1), dict(k=700), dict(k=15000), dict(p=0.2), dict(p=0.3), dict(p=0.97),
                                dict(p=0.9, mp=0.1), dict(k=2000, p=0.5), dict(T=0.05, p=0.8), dict(T=30.0, p=0.5), dict(T=1e35, p=0.5)])
@pytest.mark.parametrize("V", [15011, 20011, 30011])
def test_sample_many_rows(ctx, V, kw):
    """The forms for many rows (in shared memory or read from L2, with and without the counting pass):
    rows where the list is too short, the border lies at a bucket's end or far from where the count puts
    it, or nothing is ordinary.  20 copies of 9 rows give the same ids."""
    rng = np.random.default_rng(11)
    base = (rng.standard_normal(V) * 2.5).astype(np.float32)
    peaks = base.copy()
    peaks[rng.integers(0, V, 6)] += 14
    masked = np.where(rng.random(V) < 0.9, -np.inf, base).astype(np.float32)
    lowest = np.where(rng.random(V) < 0.5, np.finfo(np.float32).min, base).astype(np.float32)
    two = rng.integers(0, 2, V).astype(np.float32)
    pinf = base.copy()
    pinf[[3, V - 12]] = np.inf
    near = (np.round(base * 4) / 4).astype(np.float32)
    # most of the weight at one logit, half a bucket from its bucket's middle, behind a few that hold the border
    off = np.full(V, -40.0, np.float32)
    off[1:2001], off[2001:12001], off[0] = rng.uniform(-6.9, -6.1, 2000), -7.0, 0.0
    off = off[rng.permutation(V)]
    rows = np.stack([base, peaks, masked, lowest, two, pinf, near, np.zeros(V, np.float32), off])
    from voxcpm_rs_b200.sampling import sample
    args = {n: kw.get(s) for n, s in (("temperature", "T"), ("top_k", "k"), ("top_p", "p"), ("min_p", "mp"))}
    full = {n: None if v is None else _cuda(np.full(180, v, np.int32 if n == "top_k" else np.float32)) for n, v in args.items()}
    for u in (0.0, 0.4321, 0.99):
        want = [osm.sample_row(r, np.float32(u), np.float32(kw.get("T", 1.0)), kw.get("k", 0), np.float32(kw.get("p", 1.0)),
                               np.float32(kw.get("mp", 0.0)))[0] for r in rows]
        ids = sample(ctx, _cuda(np.tile(rows, (20, 1))), _cuda(np.full(180, u, np.float32)), **full).cpu().numpy()
        assert ids.reshape(20, 9).tolist() == [want] * 20, u


def test_sample_one_row_for_many_draws(ctx):
    """An expanded row (stride 0) is read by every draw; a negative stride is refused."""
    import torch
    from voxcpm_rs_b200 import _lib
    from voxcpm_rs_b200.sampling import sample
    rng = np.random.default_rng(4)
    x, u = _logits(rng, 1, 3001), rng.random(37).astype(np.float32)
    t = _cuda(x)
    ids = sample(ctx, t.expand(37, 3001), _cuda(u), top_p=_cuda(np.full(37, 0.9, np.float32)))
    assert ids.tolist() == [osm.sample_row(x[0], v, top_p=np.float32(0.9))[0] for v in u]
    assert torch.equal(ids, sample(ctx, t.repeat(37, 1), _cuda(u), top_p=_cuda(np.full(37, 0.9, np.float32))))
    L = _lib.lib()
    call = lambda stride, rows, vocab: L.vx_sample(ctx.h, t.data_ptr(), stride, rows, vocab, _cuda(u).data_ptr(), None, None,  # noqa: E731
                                                   None, None, ids.data_ptr(), None, None)
    assert [call(-1, 2, 100), call(0, -1, 100), call(0, 2 ** 20 + 1, 100), call(0, 1, 0), call(0, 1, 2 ** 18 + 1)] == [
        _lib.VX_ERR_SHAPE] * 5
