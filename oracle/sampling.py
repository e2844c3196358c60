"""Token sampling in numpy, in 64 bits: temperature, top-k, top-p, min-p, and a draw in index
order from a given random number."""
from __future__ import annotations

import numpy as np

ONE = float(1 << 44)


def sample_row(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(id, log-probability) of one row; see ``vx_sample``."""
    x = np.asarray(logits, np.float64)
    if np.isnan(x).any() or not temperature >= 0:
        return -1, np.nan
    top = x.max()
    if top == -np.inf:
        return -1, -np.inf
    if temperature == 0:
        return int(np.argmax(x)), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(x == top, 0.0, (x - top) / np.float64(temperature))
    z = np.where(np.isnan(z), -np.inf, z)  # next to +inf, or -inf itself, at an infinite temperature
    w = [int(t) for t in np.rint(np.exp(z) * ONE)]
    order = [int(i) for i in np.argsort(-x, kind="stable")]
    if 0 < top_k < len(x):
        order = order[:top_k]
    if top_p < 1:
        mass = sum(w[i] for i in order)
        need = max(1, int(np.ceil(np.float64(top_p) * np.float64(mass))))
        run, n = 0, 0
        while run < need:
            run += w[order[n]]
            n += 1
        order = order[:n]
    least = min(float(min_p), 1.0) * ONE
    stay = sorted(i for i in order if w[i] >= least)
    total = sum(w[i] for i in stay)
    at = min(int(np.floor(max(np.float64(u), 0.0) * np.float64(total))), total - 1)
    run = 0
    for i in stay:
        run += w[i]
        if run > at:
            return i, float(np.log(np.float64(w[i]) / np.float64(total)))
    raise AssertionError("no token")
