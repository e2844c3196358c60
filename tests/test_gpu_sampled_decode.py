"""The sampled decode loop of the LM, and the 4-bit cache's operators and the sampler together as a
decode loop uses them: appended, attended, evicted and drawn step by step, eagerly, in a captured
graph, and on another stream."""
import math

import numpy as np
import pytest

from oracle import kv4 as ok
from oracle import minicpm4 as om
from oracle import sampling as osm

pytestmark = pytest.mark.gpu


def _cuda(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.fixture(scope="module")
def lm(ctx):
    from tests.golden.make_golden import small_lm_config
    from voxcpm_rs_b200 import synth
    from voxcpm_rs_b200.minicpm4 import MiniCpmModel
    cfg = small_lm_config()
    w = synth.minicpm_weights(cfg, seed=5, std=0.2)
    m = MiniCpmModel(ctx, cfg, w, max_batch=4, max_length=96)
    yield cfg, m, synth.minicpm_f32_view(w)
    m.close()


def test_lm_sample_at_temperature_zero_is_greedy(lm):
    """Temperature 0, and top_k 1 at any temperature, give vx_lm_greedy's ids; rows do not mix."""
    cfg, m, _ = lm
    rng = np.random.default_rng(0)
    prompts = rng.integers(0, cfg.vocab_size, (3, 11))
    want = np.stack([m.greedy(p, 20) for p in prompts])
    u = rng.random((21, 3))
    assert np.array_equal(m.sample(prompts, 20, u, temperature=0.0), want)
    assert np.array_equal(m.sample(prompts, 20, u, temperature=1.3, top_k=1), want)
    mixed = m.sample(prompts, 20, u, temperature=[0.0, 1.0, 0.0])
    assert np.array_equal(mixed[[0, 2]], want[[0, 2]])
    one = m.sample(prompts[1], 20, u[:, 1:2], temperature=1.0)
    assert one.shape == (1, 21)
    assert np.array_equal(m.greedy(prompts[0], 20), want[0])  # the greedy path is as it was


@pytest.mark.parametrize("kw", [dict(temperature=0.8), dict(temperature=1.0, top_k=20), dict(temperature=0.7, top_p=0.9),
                                dict(temperature=1.5, min_p=0.05)])
def test_lm_sample_draws_from_the_model(lm, kw):
    """Each drawn id's interval of the running sum of the oracle's probabilities holds u.  The oracle's
    logits differ from the library's by the f32 path's 1e-3 of the largest at most, so a probability
    by exp(2e-3 max / T) - 1 relative, and so the ends of the interval and the borders of the kept set."""
    cfg, m, w = lm
    rng = np.random.default_rng(1)
    B, n, steps = 2, 9, 12
    prompts = rng.integers(0, cfg.vocab_size, (B, n))
    u = rng.random((steps + 1, B)).astype(np.float32)
    ids = m.sample(prompts, steps, u, **kw)
    T = kw["temperature"]
    for b in range(B):
        seq = np.concatenate([prompts[b], ids[b]])
        h = om.model_forward(cfg, w, om.embed(cfg, w, seq[None, :-1]), True)[0][0, n - 1:]
        logits = (h @ w["embed"].T).astype(np.float64)
        for s in range(steps + 1):
            l = logits[s]
            eps = math.exp(2e-3 * np.abs(l).max() / T) - 1
            p = np.exp((l - l.max()) / T)
            order = np.argsort(-l, kind="stable")
            # a set that surely holds what stays, and one that is surely held
            sure, may = np.ones(len(l), bool), np.ones(len(l), bool)
            if "top_k" in kw:
                edge = p[order[kw["top_k"] - 1]]
                sure, may = p > edge * (1 + eps), p >= edge * (1 - eps)
            if "top_p" in kw:
                c = np.cumsum(p[order]) / p.sum()
                sure[order], may[order] = c < kw["top_p"] - eps, c - p[order] / p.sum() < kw["top_p"] + eps
            if "min_p" in kw:
                sure, may = p >= kw["min_p"] * (1 + eps), p >= kw["min_p"] * (1 - eps)
            i = ids[b, s]
            assert may[i]
            most, least = p[may].sum() * (1 + eps), max(p[sure].sum(), p.max()) * (1 - eps)
            lo = p[:i][sure[:i]].sum() * (1 - eps) / most
            hi = (p[:i + 1][may[:i + 1]].sum()) * (1 + eps) / least
            assert lo <= u[s, b] <= hi, (b, s, lo, u[s, b], hi)


def test_lm_sample_refusals(lm):
    from voxcpm_rs_b200._lib import VX_ERR_ARG, VX_ERR_CANCELLED, VX_ERR_KV_FULL, VX_ERR_SHAPE, VxError
    cfg, m, _ = lm
    p = np.zeros((2, 5), np.int32)
    for call, code in ((lambda: m.sample(p, 92, np.zeros((93, 2))), VX_ERR_KV_FULL),
                       (lambda: m.sample(p, 3, np.zeros((3, 2))), VX_ERR_SHAPE),
                       (lambda: m.sample(np.zeros((5, 5)), 3, np.zeros((4, 5))), VX_ERR_SHAPE),
                       (lambda: m.sample(p - 1, 3, np.zeros((4, 2))), VX_ERR_ARG)):
        with pytest.raises(VxError) as e:
            call()
        assert e.value.code == code
    m.ctx.cancel()
    with pytest.raises(VxError) as e:
        m.sample(p, 3, np.zeros((4, 2)))
    assert e.value.code == VX_ERR_CANCELLED
    m.ctx.cancel_reset()
    assert m.sample(p, 91, np.zeros((92, 2))).shape == (2, 92)


# --------------------------------------------------------- the 4-bit cache and the sampler together

class Loop:
    """A decode step over one cached layer: a token's q | k | v row (a table in place of a projection),
    appended, attended with its weights, the block of least weight let go of at the budget, logits by
    a matrix, and the next token drawn.  All state is on the device, so a step can be captured."""

    def __init__(self, ctx, B=3, nkv=2, nrep=4, d=64, budget=40, block=8, vocab=500, seed=0):
        import torch
        from voxcpm_rs_b200.kv4 import Kv4Cache
        rng = np.random.default_rng(seed)
        self.B, self.nkv, self.nrep, self.d, self.budget, self.block, self.ctx = B, nkv, nrep, d, budget, block, ctx
        self.table = _cuda(rng.standard_normal((vocab, (nkv * nrep + 2 * nkv) * d)).astype(np.float32))
        self.head = _cuda((rng.standard_normal((nkv * nrep * d, vocab)) * 0.3).astype(np.float32))
        self.cache = Kv4Cache(ctx, B, nkv, budget, d)
        self.lens = torch.zeros(B, device="cuda", dtype=torch.int32)
        self.seen = torch.zeros(B, device="cuda", dtype=torch.int32)
        self.ids = torch.arange(B, device="cuda")
        self.u = torch.zeros(B, device="cuda")
        self.T = torch.full((B,), 0.7, device="cuda")
        self.top_k = torch.full((B,), 50, device="cuda", dtype=torch.int32)
        self.cap = self.cache.capacity

    def step(self, evict):
        import torch
        from voxcpm_rs_b200.sampling import sample
        nq, nk = self.nkv * self.nrep * self.d, self.nkv * self.d
        row = self.table[self.ids].unsqueeze(1)
        k, v = (row[..., nq + i * nk:nq + (i + 1) * nk].unflatten(-1, (self.nkv, self.d)) for i in range(2))
        if evict:
            self.lens.copy_(self.cache.evict(self.lens, self.seen, self.cap - self.block, sink=2, recent=6))
        self.cache.append(k, v, self.lens, first_position=self.seen)
        self.lens += 1
        self.seen += 1
        self.out = self.cache.attend(row[:, 0, :nq], self.lens, track=True)
        self.logits = self.out @ self.head
        ids = sample(self.ctx, self.logits, self.u, temperature=self.T, top_k=self.top_k)
        self.ids.copy_(ids)
        return ids, torch.clone(self.out)


def _numpy_loop(loop, table, first, evicts):
    """The same steps by the definitions in 64 bits, given the ids that were drawn."""
    B, nkv, d, nq, nk = loop.B, loop.nkv, loop.d, loop.nkv * loop.nrep * loop.d, loop.nkv * loop.d
    rows = [[[] for _ in range(nkv)] for _ in range(B)]  # [k, v, weight, position]
    ids, t = list(first), 0
    while True:
        outs = np.zeros((B, nq))
        for b in range(B):
            x = table[ids[b]]
            for h in range(nkv):
                r = rows[b][h]
                if evicts[t]:
                    w, pos = np.array([e[2] for e in r]), np.array([e[3] for e in r])
                    src = ok.evict(w.astype(np.float32), pos, len(r), t, loop.cap - loop.block, 2, 6)
                    rows[b][h] = r = [r[i] for i in src]
                k, v = (ok.values(*ok.quantise(x[nq + i * nk + h * d:nq + i * nk + (h + 1) * d][None])) [0] for i in range(2))
                r.append([k, v, 0.0, t])
                q = x[:nq].reshape(nkv, loop.nrep, d)[h][None]
                o, p = ok.attend(q, np.stack([e[0] for e in r])[None, None], np.stack([e[1] for e in r])[None, None],
                                 [len(r)], loop.nrep, 1 / math.sqrt(d))
                outs[b].reshape(nkv, loop.nrep, d)[h] = o[0]
                for e, got in zip(r, p[0, 0]):
                    e[2] += got
        t += 1
        ids = yield outs


def test_decode_loop_with_eviction_matches_the_definitions(ctx):
    """60 steps over a budget of 64 rows with blocks of 8 let go of: attention outputs as the
    definitions give them for the same ids, ids as the sampler's definition gives them for the
    step's logits.  Weights differ from the 64-bit ones by 1e-5 of a row's at most, far less than
    weights differ from one another (checked), so the same rows go."""
    import torch
    loop = Loop(ctx, budget=33)
    rng = np.random.default_rng(4)
    n = 150
    evicts, size = [], 0
    for _ in range(n):
        evicts.append(size == loop.cap)
        size = (loop.cap - loop.block if evicts[-1] else size) + 1
    us = rng.random((n, loop.B)).astype(np.float32)
    ref = _numpy_loop(loop, loop.table.cpu().numpy(), loop.ids.tolist(), evicts)
    want = next(ref)
    for t in range(n):
        loop.u.copy_(torch.from_numpy(us[t]))
        ids, out = loop.step(evicts[t])
        assert np.abs(out.cpu().numpy() - want).max() < 1e-4, t
        logits = loop.logits.cpu().numpy()
        ids = ids.tolist()
        for b in range(loop.B):
            assert ids[b] == osm.sample_row(logits[b], us[t, b], np.float32(0.7), 50)[0], (t, b)
        if t + 1 < n:
            want = ref.send(ids)
    assert loop.lens.tolist() == [size] * loop.B and loop.seen.tolist() == [n] * loop.B
    ctx.synchronize()


def test_captured_steps_replay_as_eager_ones(ctx):
    """A step with eviction and one without, each captured into a graph of its own and replayed in
    turn, on a stream of their own: bits as the eager loop's.  The graphs' workspaces are their own."""
    import torch
    a, b = Loop(ctx, seed=1), Loop(ctx, seed=1)
    us = np.random.default_rng(5).random((120, a.B)).astype(np.float32)
    warm = Loop(ctx, seed=1)
    for e in (False, True):
        warm.step(e)
    torch.cuda.synchronize()
    graphs = {}
    for e in (False, True):
        g = torch.cuda.CUDAGraph()
        state = [t.clone() for t in (b.lens, b.seen, b.ids)]
        with torch.cuda.graph(g):
            graphs[e] = (g, b.step(e))
        for t, s in zip((b.lens, b.seen, b.ids), state):
            t.copy_(s)
    side = torch.cuda.Stream()
    size = 0
    for t in range(120):
        e = size == a.cap
        size = (a.cap - a.block if e else size) + 1
        u = torch.from_numpy(us[t])
        a.u.copy_(u)
        ids, out = a.step(e)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            b.u.copy_(u)
            graphs[e][0].replay()
        torch.cuda.synchronize()
        gi, go = graphs[e][1]
        assert torch.equal(ids, gi) and torch.equal(out, go), t
    assert torch.equal(a.cache.weights, b.cache.weights) and torch.equal(a.cache.positions, b.cache.positions)
    ctx.synchronize()


def test_calls_follow_the_current_stream(ctx):
    """Calls run on the current stream: behind a long kernel on a side stream they wait for its inputs."""
    import torch
    loop, ref = Loop(ctx, seed=2), Loop(ctx, seed=2)
    for t in range(50):
        ref.step(False) if t < 40 else ref.step(ref.lens[0].item() == ref.cap)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big = torch.randn(6000, 6000, device="cuda")
        for _ in range(5):
            big = big @ big * 1e-4
        loop.u.add_(big[0, 0] * 0)  # the loop's input depends on them
        for t in range(50):
            loop.step(False) if t < 40 else loop.step(loop.lens[0].item() == loop.cap)
    side.synchronize()
    assert torch.equal(loop.ids, ref.ids) and torch.equal(loop.out, ref.out)


def test_tracking_does_not_change_the_output_or_the_cache(ctx):
    """Long and short caches, with and without track: the same bits; rows are only read."""
    import torch
    from tests.test_gpu_kv4 import _filled, _raw
    rng = np.random.default_rng(6)
    for n, nrep in ((100, 8), (6000, 8), (500, 12)):
        c, _, _ = _filled(ctx, rng, 2, 2, n, 128)
        q = _cuda(rng.standard_normal((2, 2 * nrep * 128)).astype(np.float32))
        lens = _cuda(np.array([n, n // 3], np.int32))
        before = _raw(c)
        assert torch.equal(c.attend(q, lens), c.attend(q, lens, track=True))
        assert all(np.array_equal(x, y) for x, y in zip(before, _raw(c)))
        # each row of the batch gave its query heads' probabilities: nrep per KV head
        s = c.weights.double().sum(-1)
        assert (s - nrep).abs().max() < nrep * (n + 300) * 2.0 ** -24 + 1e-5


def test_offsets_past_32_bits(ctx):
    """A cache whose code buffers pass 2^31 bytes: append, read, attention and eviction of its last
    sequence agree with a small cache's."""
    import torch
    from voxcpm_rs_b200.kv4 import Kv4Cache
    nkv, d, cap, B = 8, 128, 131072, 33  # 2.2 GB of codes for K, as much for V
    big, small = Kv4Cache(ctx, B, nkv, cap, d), Kv4Cache(ctx, 1, nkv, cap, d)
    rng = np.random.default_rng(7)
    n = 3000
    x = _cuda(rng.standard_normal((1, n, 2 * nkv * d)).astype(np.float32))
    k, v = (x[..., i * nkv * d:(i + 1) * nkv * d].unflatten(-1, (nkv, d)) for i in range(2))
    z = lambda val: torch.zeros(B, device="cuda", dtype=torch.int32).index_fill_(0, torch.tensor([B - 1], device="cuda"), val)  # noqa: E731
    at = cap - n
    one = lambda val: torch.full((1,), val, device="cuda", dtype=torch.int32)  # noqa: E731
    big.append(k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), z(at), z(n))
    small.append(k, v, one(at))
    # the rows of the whole last sequence, zeros first
    q = _cuda(rng.standard_normal((1, nkv * 8 * d)).astype(np.float32))
    a = big.attend(q.expand(B, -1), z(cap), track=True)
    b = small.attend(q, one(cap), track=True)
    assert torch.allclose(a[-1], b[0], rtol=0, atol=1e-5) and (a[:-1] == 0).all()
    assert torch.allclose(big.weights[-1], small.weights[0], rtol=0, atol=1e-5)
    small.weights.copy_(big.weights[-1:])
    la = big.evict(z(cap), z(cap), 4096, 4, 100)
    lb = small.evict(one(cap), one(cap), 4096, 4, 100)
    assert la[-1] == 4096 and lb[0] == 4096 and (la[:-1] == 0).all()
    ka, kb = big.read(4096, counts=la)[0], small.read(4096, counts=lb)[0]
    assert torch.equal(ka[-1], kb[0]) and torch.equal(big.positions[-1, :, :4096], small.positions[0, :, :4096])
    ctx.synchronize()
