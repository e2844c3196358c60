"""The 4-bit KV cache in numpy, in 64 bits: the row format, append, attention and eviction as
their definitions say, row by row."""
from __future__ import annotations

import numpy as np

CODE_VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def e4m3_values():
    """The 127 non-negative finite e4m3 numbers by bit pattern."""
    b = np.arange(127)
    e, m = b >> 3, b & 7
    return np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))


def _nearest_even(y, table):
    """Index of the nearest entry of an ascending table, ties to the even index, clamped."""
    hi = np.clip(np.searchsorted(table, y), 1, len(table) - 1)
    a, b = y - table[hi - 1], table[hi] - y
    return np.where((b < a) | ((a == b) & (hi % 2 == 0)), hi, hi - 1)


def quantise(x):
    """``x [..., d]`` f32 -> (codes uint8 ``[..., d/2]``, scale bytes uint8 ``[..., d/16]``)."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 16)
    amax = np.abs(g).max(-1)
    bad = np.isnan(amax)
    table = e4m3_values()
    s8 = _nearest_even(np.minimum(np.where(bad, 0.0, amax) / 6.0, 448.0), table)
    s = table[s8][..., None]
    with np.errstate(invalid="ignore", divide="ignore"):
        y = np.where(s > 0, np.abs(g) / np.where(s > 0, s, 1.0), 0.0)
    code = _nearest_even(np.minimum(np.nan_to_num(y, nan=0.0, posinf=6.0), 6.0), CODE_VALUES)
    code = (code | (np.signbit(g).astype(int) << 3)).reshape(*x.shape[:-1], -1, 2)
    return ((code[..., 0] | (code[..., 1] << 4)).astype(np.uint8),
            np.where(bad, 127, s8).astype(np.uint8))


def values(codes, scales):
    """The numbers that rows of codes and scale bytes stand for."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])
    v = np.concatenate([CODE_VALUES, -CODE_VALUES])[c]
    s = np.append(e4m3_values(), np.nan)[scales & 127]
    return (v.reshape(*s.shape, 16) * s[..., None]).reshape(v.shape)


def attend(q, k, v, lens, nrep, scale):
    """q ``[B, nh, d]``, k, v ``[B, nkv, n, d]`` values: out ``[B, nh, d]`` and the probabilities that
    each row received ``[B, nkv, n]``."""
    B, nkv, n, d = k.shape
    out, got = np.zeros(q.shape), np.zeros((B, nkv, n))
    for b in range(B):
        m = int(lens[b])
        if m == 0:
            continue
        for h in range(q.shape[1]):
            g = h // nrep
            s = k[b, g, :m] @ q[b, h].astype(np.float64) * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[b, h] = p @ v[b, g, :m]
            got[b, g, :m] += p
    return out, got


def evict(weights, positions, length, seen, keep, sink, recent):
    """Of one KV head: the row that each slot below the new length takes."""
    w, pos = np.asarray(weights[:length], np.float64), positions[:length]
    if length <= keep:
        return np.arange(length)
    safe = (pos < sink) | (pos >= seen - recent)
    # rank: protected rows, then NaN, then the larger weight; the lower slot first
    order = np.lexsort((np.arange(length), -np.nan_to_num(w, nan=0.0, posinf=np.inf), ~np.isnan(w), ~safe))
    order = np.concatenate([np.flatnonzero(safe), order[~safe[order]]])
    kept = np.zeros(length, bool)
    kept[order[:keep]] = True
    src = np.arange(keep)
    src[~kept[:keep]] = keep + np.flatnonzero(kept[keep:])
    return src
