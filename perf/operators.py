"""Cases of the 4-bit KV cache and token sampling operators: what is measured, in plain torch and through
this package's own kernels.

Cache rows.  A key or value row of ``d`` numbers is held as ``d / 2`` bytes of e2m1 codes (dim 2j in the low
nibble of byte j) and ``d / 16`` e4m3 scales, one for each 16 dims: value = code value * scale.

Operators (``case["op"]``)
  append   rows of new tokens quantised into the cache, and the values that they then stand for
  attend   one query token of each sequence over its cached rows; with ``track`` the probability that each
           row received, summed over the query heads that share it, is added to the row's running weight
  evict    the ``keep`` rows of largest weight stay (the first ``sink`` positions and the last ``recent`` ones
           always do); kept rows behind slot ``keep`` move into the slots that became free
  sample   one token id of each row of logits: temperature, top-k, top-p, min-p, and a draw from a given u
"""
import math

import torch

own = False

_CODE_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# |x| / scale at which e2m1 goes from one code to the next; a tie goes to the code whose last bit is 0
_CODE_EDGES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)
_WEIGHT_BITS = 44  # a token's weight exp(.) is taken to so many binary places

_contexts = {}


def _context():
    """One library context of the current device, as a program keeps it."""
    from __graft_entry__ import load_package
    load_package()
    from voxcpm_rs_b200.minicpm4 import Context
    i = torch.cuda.current_device()
    if i not in _contexts:
        _contexts[i] = Context(i)
    return _contexts[i]


def listed():
    return [
        # one decoded token of 8 utterances goes into the cache (the decoder's 2 KV heads of 128)
        dict(name="append_token", op="append", B=8, S=1, nkv=2, d=128, cap=4096, ragged=True),
        # ragged prompts of a batch are written in one call (the decoder's heads)
        dict(name="append_prompts", op="append", B=16, S=4093, nkv=2, d=128, cap=8192, ragged=True),
        # one utterance, the decoder's 16 query heads over 2 KV heads, a short cache
        dict(name="attend_one", op="attend", B=1, nkv=2, nrep=8, d=128, max_len=1001, ragged=False, track=False),
        # one long document's cache: few heads, the long axis has to be split
        dict(name="attend_long", op="attend", B=1, nkv=2, nrep=8, d=128, max_len=131071, ragged=False, track=False),
        # a ragged batch that keeps the running weights for eviction
        dict(name="attend_track", op="attend", B=32, nkv=2, nrep=8, d=128, max_len=8191, ragged=True, track=True),
        # the 64-wide heads of the diffusion stack, 7 query heads to a KV head
        dict(name="attend_d64", op="attend", B=24, nkv=4, nrep=7, d=64, max_len=4097, ragged=True, track=True),
        # a full serving batch of long sequences
        dict(name="attend_full", op="attend", B=64, nkv=2, nrep=8, d=128, max_len=32768, ragged=False, track=False),
        # a decode loop at its budget lets go of a block of rows
        dict(name="evict_block", op="evict", B=8, nkv=2, d=128, max_len=4160, keep=4096, sink=4, recent=256, ragged=False),
        # long prompts are cut down to a decode budget
        dict(name="evict_prompts", op="evict", B=16, nkv=2, d=128, max_len=32749, keep=2048, sink=4, recent=512, ragged=True),
        # one utterance's next token at the model's vocabulary
        dict(name="sample_one", op="sample", rows=1, vocab=73448, mix="topk"),
        # a serving batch whose requests each have their own settings
        dict(name="sample_batch", op="sample", rows=64, vocab=73448, mix="all"),
        # nucleus sampling alone, a larger odd vocabulary, many rows
        dict(name="sample_nucleus", op="sample", rows=256, vocab=151643, mix="topp"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "evict", "sample"])
    d = rng.choice([64, 128, 128])
    if op == "append":
        B, S = _log_int(rng, 1, 32), _log_int(rng, 1, 4096)
        nkv = rng.choice([1, 2, 4, 8])
        while B * S * nkv > 16 * 8192:
            B, S = max(1, B // 2), max(1, S // 2 + 1)
            nkv = max(1, nkv // 2)
        return dict(op=op, B=B, S=S, nkv=nkv, d=d, cap=S + rng.randint(1, 4096), ragged=rng.random() < 0.7)
    if op == "attend":
        B, nkv = _log_int(rng, 1, 64), rng.choice([1, 2, 2, 4, 8])
        most = max(1, min(131072, 2000000 // (B * nkv)))
        return dict(op=op, B=B, nkv=nkv, nrep=rng.choice([1, 2, 4, 5, 7, 8, 8, 16]), d=d, max_len=_log_int(rng, 1, most),
                    ragged=rng.random() < 0.6, track=rng.random() < 0.5)
    if op == "evict":
        B, nkv = _log_int(rng, 1, 32), rng.choice([1, 2, 4])
        n = _log_int(rng, 2, max(2, min(131072, 1000000 // (B * nkv))))
        keep = rng.randint(1, n)
        sink = rng.randint(0, min(8, keep))
        return dict(op=op, B=B, nkv=nkv, d=d, max_len=n, keep=min(keep, 16384), sink=min(sink, 16384),
                    recent=rng.randint(0, min(keep, 16384) - sink), ragged=rng.random() < 0.6)
    return dict(op=op, rows=_log_int(rng, 1, 256), vocab=_log_int(rng, 32, 151643), mix=rng.choice(["topk", "topp", "minp", "all"]))


# ----------------------------------------------------------------------------------------------- the 4-bit rows


def _quantise(x):
    """f32 [..., d] -> (codes uint8 [..., d / 2], scales f32 [..., d / 16] on the e4m3 grid).

    The scale is amax / 6 of 16 dims rounded to e4m3 (nearest, ties to even, at most 448); a code is
    x / scale rounded to e2m1 (nearest, ties to even, at most 6)."""
    g = x.unflatten(-1, (-1, 16))
    s = (g.abs().amax(-1) / 6.0).clamp_max(448.0).to(torch.float8_e4m3fn).float()
    y = g.abs().double() / torch.where(s == 0, math.inf, s).double().unsqueeze(-1)
    code = torch.bucketize(y, _edges(x.device)) | (torch.signbit(g).long() << 3)
    code = code.to(torch.uint8).flatten(-2).unflatten(-1, (-1, 2))
    return code[..., 0] | (code[..., 1] << 4), s


def _edges(device):
    """Where a code begins, in 64 bits: just behind an edge whose tie stays below, just before one whose tie goes up."""
    t = torch.tensor(_CODE_EDGES, device=device, dtype=torch.float64)
    up = torch.tensor([0, 1, 0, 1, 0, 1, 0], device=device, dtype=torch.bool)
    return torch.where(up, torch.nextafter(t, torch.zeros_like(t)), t)


def _table(device, dtype):
    t = torch.tensor(_CODE_VALUES, device=device, dtype=dtype)
    return torch.cat([t, -t])


def _values(codes, scales, dtype=torch.float32):
    """The numbers that cache rows stand for."""
    t = _table(codes.device, dtype)
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    v = t[c.to(torch.int64)]
    s = scales.to(torch.float32).to(dtype)
    return (v.unflatten(-1, (s.shape[-1], 16)) * s.unsqueeze(-1)).flatten(-2)


def _rows(gen, shape, spread):
    """Keys or values as a model has them: unit rows with a few strong channels."""
    x = torch.randn(shape, generator=gen, device="cuda")
    strong = 1.0 + 3.0 * (torch.rand(shape[-1], generator=gen, device="cuda") < 0.06).float()
    return x * strong * spread


def _cache(gen, B, nkv, cap, d):
    """Buffers of a cache that holds rows already."""
    bufs = []
    for spread in (1.0, 0.4):
        codes = torch.empty(B, nkv, cap, d // 2, device="cuda", dtype=torch.uint8)
        scales = torch.empty(B, nkv, cap, d // 16, device="cuda", dtype=torch.float8_e4m3fn)
        some = _rows(gen, (min(cap, 2048), d), spread)
        c, s = _quantise(some)
        # rows of different sequences are different ones: a pool of quantised rows, indexed at random
        for b in range(B):
            at = torch.randint(0, some.shape[0], (nkv, cap), generator=gen, device="cuda")
            codes[b] = c[at]
            scales[b] = s[at].to(torch.float8_e4m3fn)
        bufs += [codes, scales]
    return bufs


def _lens(gen, B, most, ragged, least=0):
    if not ragged:
        return torch.full((B,), most, device="cuda", dtype=torch.int32)
    n = torch.randint(least, most + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
    n[B // 2] = most
    return n


def _round_up(n, m):
    return -(-n // m) * m


def _handle(st):
    from voxcpm_rs_b200.kv4 import Kv4Cache
    return Kv4Cache.from_buffers(_context(), *st["bufs"], weights=st.get("weights"), positions=st.get("positions"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)
    op, st = case["op"], dict(case)
    if own:
        _context()
    if op == "sample":
        R, V = case["rows"], case["vocab"]
        x = torch.randn(R, V, generator=gen, device="cuda") * 2.5
        peak = torch.randint(0, V, (R, 12), generator=gen, device="cuda")
        x.scatter_add_(1, peak, torch.rand(R, 12, generator=gen, device="cuda") * 9.0)
        x[torch.rand(R, V, generator=gen, device="cuda") < 0.01] = -math.inf  # tokens that may not come
        st["logits"] = x
        st["u"] = torch.rand(R, generator=gen, device="cuda")
        r = torch.rand(4, R, generator=gen, device="cuda")
        mix = case["mix"]
        st["temperature"] = 0.6 + 0.6 * r[0]
        if mix == "all":
            st["temperature"] = torch.where(r[0] < 0.1, torch.zeros_like(r[0]), st["temperature"])  # some are greedy
        st["top_k"] = (1 + (r[1] * 100)).to(torch.int32) if mix in ("topk", "all") else None
        if mix == "all":
            st["top_k"] = torch.where(r[1] < 0.4, torch.zeros_like(st["top_k"]), st["top_k"])  # 0: no limit
        st["top_p"] = 0.8 + 0.19 * r[2] if mix in ("topk", "topp", "all") else None
        st["min_p"] = 0.02 + 0.1 * r[3] if mix in ("minp", "all") else None
        if mix == "all":
            st["min_p"] = torch.where(r[3] < 0.5, torch.zeros_like(r[3]), st["min_p"])
        return st
    B, nkv, d = case["B"], case["nkv"], case["d"]
    if op == "append":
        S, cap = case["S"], _round_up(case["cap"], 32)
        # keys and values come out of a fused projection: rows of q | k | v
        wide = _rows(gen, (B, S, 2 * nkv * d), 1.0)
        st["k"] = wide[..., : nkv * d].unflatten(-1, (nkv, d))
        st["v"] = wide[..., nkv * d:].unflatten(-1, (nkv, d))
        st["bufs"] = _cache(gen, B, nkv, 32, d)
        st["bufs"] = [t.repeat(1, 1, cap // 32, 1) for t in st["bufs"]]
        st["counts"] = _lens(gen, B, S, case["ragged"])
        room = cap - S
        st["start"] = torch.randint(0, room + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
    else:
        n = case["max_len"]
        cap = _round_up(n, 32)
        st["bufs"] = _cache(gen, B, nkv, cap, d)
        st["lens"] = _lens(gen, B, n, case["ragged"])
        if op == "attend":
            st["q"] = torch.randn(B, nkv * case["nrep"] * d, generator=gen, device="cuda")
            if case["track"]:
                st["weights"] = torch.rand(B, nkv, cap, generator=gen, device="cuda")
        else:
            # running weights as attention leaves them: most rows little, a few much
            st["weights"] = torch.rand(B, nkv, cap, generator=gen, device="cuda").pow_(6) * 20
            slots = torch.arange(cap, device="cuda", dtype=torch.int32)
            st["positions"] = (slots + (slots >= 64) * 100).expand(B, nkv, cap).contiguous()  # 100 tokens went before
            st["seen"] = st["lens"] + 100
            st["weights_out"] = torch.zeros_like(st["weights"])
            st["positions_out"] = torch.zeros_like(st["positions"])
    if own:
        st["cache"] = _handle(st)
    return st


# ------------------------------------------------------------------------------------------------- the passes


def run(st):
    op = st["op"]
    if own:
        return _own(st)
    if op == "append":
        return _plain_append(st)
    if op == "attend":
        return _plain_attend(st)
    if op == "evict":
        return _plain_evict(st)
    return _plain_sample(st["logits"], st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"])


def _own(st):
    op = st["op"]
    if op == "sample":
        from voxcpm_rs_b200.sampling import sample
        ids, logprob = sample(_context(), st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"],
                              top_p=st["top_p"], min_p=st["min_p"], return_logprob=True)
        return {"ids": ids, "logprob": logprob}
    cache = st["cache"]
    if op == "append":
        cache.append(st["k"], st["v"], st["start"], st["counts"])
        k, v = cache.read(st["S"], start=st["start"], counts=st["counts"])
        return {"k": k, "v": v}
    if op == "attend":
        out = cache.attend(st["q"], st["lens"], st["max_len"], track=st["track"])
        return {"out": out, "weights": cache.weights} if st["track"] else {"out": out}
    lens = cache.evict(st["lens"], st["seen"], st["keep"], sink=st["sink"], recent=st["recent"], max_len=st["max_len"],
                       weights_out=st["weights_out"], positions_out=st["positions_out"])
    k, v = cache.read(min(st["keep"], st["max_len"]), counts=lens)
    return {"lens": lens, "weights": st["weights_out"], "positions": st["positions_out"], "k": k, "v": v}


def _plain_append(st):
    B, S, nkv, d = st["k"].shape
    i = torch.arange(S, device="cuda")
    there = i[None, :] < st["counts"][:, None]
    slot = (st["start"][:, None] + i[None, :]).long()
    b = torch.arange(B, device="cuda")[:, None].expand(B, S)[there]
    at = slot[there]
    got = {}
    for name, x, codes, scales in (("k", st["k"], *st["bufs"][:2]), ("v", st["v"], *st["bufs"][2:])):
        c, s = _quantise(x)
        codes[b, :, at] = c[there]
        scales.view(torch.uint8)[b, :, at] = s[there].to(torch.float8_e4m3fn).view(torch.uint8)
        bb = torch.arange(B, device="cuda")[:, None]
        y = _values(codes[bb, :, slot], scales.view(torch.uint8)[bb, :, slot].view(torch.float8_e4m3fn))
        got[name] = torch.where(there[:, :, None, None], y, 0.0).transpose(1, 2).contiguous()
    return got


def _attend(q, bufs, lens, n):
    """out [B, nh d] and the probabilities that each row received."""
    B, nkv = bufs[0].shape[:2]
    d = bufs[0].shape[3] * 2
    k, v = _values(bufs[0][:, :, :n], bufs[1][:, :, :n]), _values(bufs[2][:, :, :n], bufs[3][:, :, :n])
    qh = q.view(B, nkv, -1, d)
    s = torch.einsum("bhrd,bhnd->bhrn", qh, k) / math.sqrt(d)
    there = (torch.arange(n, device=q.device)[None, :] < lens[:, None])[:, None, None, :]
    s = torch.where(there, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0, 1.0, l)
    out = torch.einsum("bhrn,bhnd->bhrd", p, v).reshape(B, -1)
    return out, p.sum(2)


def _plain_attend(st):
    n = st["max_len"]
    tf32 = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    B, nkv, d = st["B"], st["nkv"], st["d"]
    some = max(1, int(1.5e9) // (nkv * n * d * 4))  # sequences whose rows are laid out in full at a time
    outs = [_attend(st["q"][i:i + some], [t[i:i + some] for t in st["bufs"]], st["lens"][i:i + some], n)
            for i in range(0, B, some)]
    torch.backends.cuda.matmul.allow_tf32 = tf32
    out = torch.cat([o for o, _ in outs])
    if not st["track"]:
        return {"out": out}
    st["weights"][:, :, :n] += torch.cat([w for _, w in outs])
    return {"out": out, "weights": st["weights"]}


def _chosen(weights, positions, lens, seen, n, keep, sink, recent):
    """Which slots stay (truth values [B, nkv, n])."""
    slots = torch.arange(n, device=weights.device)
    there = (slots[None, :] < lens[:, None])[:, None, :]
    w, pos = weights[:, :, :n], positions[:, :, :n]
    safe = (pos < sink) | (pos >= (seen[:, None, None] - recent))
    rank = torch.where(there, torch.where(safe, math.inf, w), -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    stays = torch.zeros(rank.shape, device=rank.device, dtype=torch.bool)
    stays.scatter_(-1, order[..., :keep], True)
    return stays & there


def _plain_evict(st):
    n, keep = st["max_len"], min(st["keep"], st["max_len"])
    w, pos = st["weights"], st["positions"]
    stays = _chosen(w, pos, st["lens"], st["seen"], n, keep, st["sink"], st["recent"])
    over = st["lens"] > keep
    hole = ~stays[..., :keep] & over[:, None, None]
    # the i-th free slot takes the i-th kept row behind slot `keep`
    mover = stays.clone()
    mover[..., :keep] = False
    src = torch.arange(keep, device="cuda").expand(*hole.shape).clone()
    src[hole] = mover.nonzero()[:, 2]
    lens = torch.minimum(st["lens"], torch.full_like(st["lens"], keep))
    there = (torch.arange(keep, device="cuda")[None, :] < lens[:, None])[:, None, :]
    for t in st["bufs"]:
        raw = t.view(torch.uint8)
        raw[:, :, :keep] = torch.gather(raw, 2, src[..., None].expand(-1, -1, -1, raw.shape[-1]))
    for a, o in ((w, st["weights_out"]), (pos, st["positions_out"])):
        o[:, :, :keep] = torch.where(there, torch.gather(a, 2, src), o[:, :, :keep])
    f = there[..., None]
    k, v = (torch.where(f, _values(st["bufs"][i][:, :, :keep], st["bufs"][i + 1][:, :, :keep]), 0.0) for i in (0, 2))
    return {"lens": lens, "weights": st["weights_out"], "positions": st["positions_out"], "k": k, "v": v}


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    R, V = logits.shape
    greedy = temperature == 0
    T = torch.where(greedy, 1.0, temperature).double()
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    one = float(1 << _WEIGHT_BITS)
    w = torch.round(torch.exp(torch.where(x == top, 0.0, (x - top) / T[:, None])) * one).long()
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices
    ws = torch.gather(w, 1, order)
    rank = torch.arange(V, device=logits.device)
    limit = torch.full((R,), V, device=logits.device, dtype=torch.int64)
    if top_k is not None:
        limit = torch.where(top_k > 0, top_k.long().clamp_max(V), limit)
    limit = torch.where(greedy, 1, limit)
    kept = rank[None, :] < limit[:, None]
    if top_p is not None:
        wk = ws * kept
        cum = wk.cumsum(-1)
        need = torch.ceil(top_p.double() * cum[:, -1].double()).long().clamp_min(1)
        kept &= torch.where(top_p[:, None] < 1, cum - wk < need[:, None], True)
    if min_p is not None:
        kept &= ws.double() >= (min_p.double().clamp_max(1.0) * one)[:, None]
    stays = torch.zeros_like(kept).scatter_(1, order, kept)
    wi = w * stays
    cum = wi.cumsum(-1)
    total = cum[:, -1]
    at = torch.floor(u.double() * total.double()).long().clamp_min(0)
    at = torch.minimum(at, total - 1)
    ids = (cum <= at[:, None]).sum(-1)
    ids = ids.clamp_max(V - 1)
    picked = torch.gather(w, 1, ids[:, None])[:, 0]
    return {"ids": ids.to(torch.int32), "logprob": torch.log(picked.double() / total.double()).float()}


# --------------------------------------------------------------------------------------------- work and exact


def work(case):
    op = case["op"]
    if op == "sample":
        R, V = case["rows"], case["vocab"]
        return {"bytes": R * V * 4 + R * 28, "flops": R * V * 4}
    B, nkv, d = case["B"], case["nkv"], case["d"]
    row = 2 * (d // 2 + d // 16)  # a cached position of one head, key and value
    mean = 0.5 if case["ragged"] else 1.0
    if op == "append":
        rows = B * case["S"] * nkv * mean
        return {"bytes": rows * (2 * d * 4 + row) + B * case["S"] * nkv * 2 * d * 4, "flops": rows * 2 * d * 4}
    rows = B * nkv * case["max_len"] * mean
    if op == "attend":
        nh = nkv * case["nrep"]
        return {"bytes": rows * (row + (8 if case["track"] else 0)) + 2 * B * nh * d * 4, "flops": rows * case["nrep"] * d * 4}
    kept = B * nkv * min(case["keep"], case["max_len"])
    return {"bytes": rows * 8 + kept * (row * 2 + 8 + 2 * d * 4), "flops": rows * 4}


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "sample":
        return _exact_sample(st)
    if op == "append":
        return {n: _exact_rows(st[n], st["counts"]) for n in ("k", "v")}
    if op == "evict":
        return _exact_evict(st)
    outs, weights = [], st["weights"].double() if case["track"] else None
    for b in range(case["B"]):  # one sequence at a time, over its own rows alone
        m = int(st["lens"][b])
        k, v = (_values(st["bufs"][i][b, :, :m], st["bufs"][i + 1][b, :, :m], torch.float64) for i in (0, 2))
        q = st["q"][b].double().view(case["nkv"], case["nrep"], case["d"])
        if m == 0:
            outs.append(torch.zeros(q.numel(), device="cuda", dtype=torch.float64))
            continue
        p = torch.softmax(q @ k.transpose(1, 2) * case["d"] ** -0.5, -1)
        outs.append((p @ v).flatten())
        if case["track"]:
            weights[b, :, :m] += p.sum(1)
    return {"out": torch.stack(outs), "weights": weights} if case["track"] else {"out": torch.stack(outs)}


def _exact_rows(x, counts):
    """The quantised rows' values: every number to the nearest of a group's 15 multiples, by distance."""
    grid = torch.arange(0, 127, device=x.device)
    e, m = (grid >> 3).double(), (grid & 7).double()
    grid = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e - 10))  # every e4m3 number, in order
    levels = torch.tensor(_CODE_VALUES, device=x.device, dtype=torch.float64)

    def nearest(y, table):  # ties to the even place in the table
        hi = torch.searchsorted(table, y).clamp(1, len(table) - 1)
        a, b = y - table[hi - 1], table[hi] - y
        return table[torch.where((b < a) | ((a == b) & (hi % 2 == 0)), hi, hi - 1)]

    y = x.double().unflatten(-1, (-1, 16))
    s = nearest((y.abs().amax(-1) / 6).contiguous(), grid).unsqueeze(-1)
    z = nearest((y.abs() / torch.where(s == 0, 1.0, s)).contiguous(), levels)
    z = torch.where(s == 0, 0.0, torch.sign(y) * z * s).flatten(-2)
    there = torch.arange(x.shape[1], device=x.device)[None, :] < counts[:, None]
    return torch.where(there[:, :, None, None], z, 0.0).transpose(1, 2).contiguous()


def _exact_evict(st):
    n, keep = st["max_len"], min(st["keep"], st["max_len"])
    B, nkv = st["weights"].shape[:2]
    wo = st["weights_out"].double()
    vals = [torch.zeros(B, nkv, keep, st["d"], device="cuda", dtype=torch.float64) for _ in range(2)]
    pool = [(st["bufs"][i], st["bufs"][i + 1]) for i in (0, 2)]
    w_all, p_all = st["weights"].cpu().numpy(), st["positions"].cpu().numpy()
    lens, seen = st["lens"].tolist(), st["seen"].tolist()
    import numpy as np
    for b in range(B):
        for h in range(nkv):
            m = lens[b]
            src = np.arange(min(m, keep))
            if m > keep:
                safe = (p_all[b, h, :m] < st["sink"]) | (p_all[b, h, :m] >= seen[b] - st["recent"])
                key = np.where(safe, np.inf, w_all[b, h, :m].astype(np.float64))
                best = np.lexsort((np.arange(m), -key))[:keep]
                kept = np.zeros(m, bool)
                kept[best] = True
                src[~kept[:keep]] = keep + np.flatnonzero(kept[keep:])
            at = torch.from_numpy(src).cuda()
            wo[b, h, :len(src)] = st["weights"][b, h, at].double()
            for t, (c, s) in zip(vals, pool):
                t[b, h, :len(src)] = _values(c[b, h, at], s[b, h].view(torch.uint8)[at].view(torch.float8_e4m3fn), torch.float64)
    return {"lens": None, "weights": wo, "positions": None, "k": vals[0], "v": vals[1]}


def _exact_sample(st):
    """The log-probability of each row's token, found by walking a sorted row."""
    import numpy as np
    if st["rows"] * st["vocab"] > 40e6:
        return None
    x_all = st["logits"].double().cpu().numpy()
    get = lambda n: None if st[n] is None else st[n].double().cpu().numpy()  # noqa: E731
    T, k, p, mp, u = (get(n) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
    out = np.zeros(len(u))
    for r, x in enumerate(x_all):
        if T[r] == 0:
            continue
        w = np.exp((x - x.max()) / T[r])
        order = np.argsort(-x, kind="stable")
        if k is not None and k[r] > 0:
            order = order[:int(k[r])]
        if p is not None and p[r] < 1:
            c = np.cumsum(w[order])
            order = order[:int(np.searchsorted(c, p[r] * c[-1])) + 1]
        if mp is not None:
            order = order[w[order] >= min(mp[r], 1.0)]
        order = np.sort(order)
        c = np.cumsum(w[order])
        i = min(int(np.searchsorted(c, u[r] * c[-1], side="right")), len(order) - 1)
        out[r] = np.log(w[order[i]] / c[-1])
    return {"ids": None, "logprob": torch.from_numpy(out)}

