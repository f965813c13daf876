"""Routing and its gradient in 64 bits, one token at a time, for the tests."""
from __future__ import annotations

import numpy as np

FLOOR = 6.103515625e-5


def scores(z, score):
    """Scores of one row (0 for an expert that takes no part), which experts take part, and whether the row has any."""
    live = ~(np.isnan(z) | (z == -np.inf))
    s = np.zeros(len(z))
    if score == "sigmoid":
        with np.errstate(over="ignore"):
            s[live] = 1.0 / (1.0 + np.exp(-z[live]))
        return s, live
    if not live.any() or z[live].max() == np.inf:
        return s, np.zeros(len(z), bool)
    e = np.exp(z[live] - z[live].max())
    s[live] = e / e.sum()
    return s, live


def pick(z, k, score="softmax", bias=None, n_group=1, topk_group=1, group_top=1):
    """The picked ids of one row, -1 where none is left."""
    s, live = scores(z, score)
    with_bias = s if bias is None else s + bias
    c = z if bias is None else with_bias
    live = live & ~np.isnan(c) & (c > -np.inf)
    if n_group > 1:
        size = len(z) // n_group
        value = np.full(n_group, -np.inf)
        for g in range(n_group):
            own = np.flatnonzero(live[g * size:(g + 1) * size]) + g * size
            if len(own):
                ranked = np.sort((with_bias if group_top == 2 else c)[own])[::-1]
                value[g] = ranked[:group_top].sum()
        kept = sorted(range(n_group), key=lambda g: (-value[g], g))[:topk_group]
        live = live & np.isin(np.arange(len(z)) // size, kept)
    order = sorted(np.flatnonzero(live), key=lambda e: (-c[e], e))[:k]
    return np.array(order + [-1] * (k - len(order)), np.int64)


def weights(z, ids, score="softmax", norm=True, scale=1.0, floor=FLOOR):
    s, _ = scores(z, score)
    w = np.where(ids < 0, 0.0, s[np.maximum(ids, 0)])
    return scale * (w / max(w.sum(), floor) if norm else w)


def gradient(z, ids, dw, score="softmax", norm=True, scale=1.0, floor=FLOOR):
    """dlogits of one row, and the sum of the magnitudes that each value is made of (what roundings are relative to)."""
    s, live = scores(z, score)
    on = (ids >= 0) & (ids < len(z))
    on[on] = live[ids[on]]
    sel = np.where(on, s[np.where(on, ids, 0)], 0.0)
    dw = np.where(on, dw, 0.0)
    S = sel.sum()
    if norm and S > floor:
        ds = scale / S * (dw - (dw * sel).sum() / S)
        mag = scale / S * (np.abs(dw) + (np.abs(dw) * sel).sum() / S)
    else:
        ds = scale * dw / (floor if norm else 1.0)
        mag = np.abs(ds)
    at, at_mag = np.zeros(len(z)), np.zeros(len(z))
    np.add.at(at, ids[on], ds[on])
    np.add.at(at_mag, ids[on], np.abs(mag[on]))
    if score == "sigmoid":
        with np.errstate(over="ignore"):
            e = np.exp(-np.abs(np.where(live, z, 0.0)))
        slope = np.where(live, e / (1.0 + e) ** 2, 0.0)
        return at * slope, at_mag * slope
    return s * (at - (at * s).sum()), s * (at_mag + (at_mag * s).sum())


def rel_tolerance(z):
    """Relative bound of an fp32 score and what is made of a few: the exponent's argument rounds to half a step of its size
    (2^-24 each), and exp, sum, quotient and products to a step or two each."""
    live = z[np.isfinite(z)]
    span = min(float(live.max() - live.min()), 104.0) if len(live) else 0.0
    return (4.0 * span + 80.0) * 2.0 ** -24
