"""The answers that the sampler's definition leaves open: of each row the first and the last
place, in the order of its logits, that a draw may come to.

A weight of the kernel is a whole number of 2^-42 of the row's largest: within 2^-43 of its
own value, and it may count as 0 below 2^-44.  Sums of V of them (C_1 = 1) are within
V 2^-43, their division among bins adds a rounding of float64 for each of 1024, so cuts and
draws are the definition's with bounds moved by at most TOL = (V + 1) 2^-41 of the sum,
and a weight meets min_p within 2^-42.  prob is w / C_n for an n between the cuts' two ends.
"""
from __future__ import annotations

import numpy as np


def place_range(x, t, k, p, m, u):
    """float64 logits x: (order, weights in it, their sums, least and most n, least and most
    place); t > 0 and at least one finite logit."""
    order = np.argsort(-x, kind="stable")
    xs = x[order]
    with np.errstate(invalid="ignore"):
        w = np.where(xs == xs[0], 1.0, np.exp((xs - xs[0]) / max(t, 2.0 ** -14)))
    c = np.cumsum(w)
    V = len(x)
    tol = (V + 1) * 2.0 ** -41

    def count(upto, bound, move):  # how many of the first `upto` sums are below the bound
        return int(np.searchsorted(c[:upto], bound + move * tol * max(bound, 1.0)))

    nk = min(k, V) if k > 0 else V
    least = most = nk
    if p < 1:
        bound = p * c[nk - 1]
        least = min(least, count(nk, bound, -1) + 1)
        most = min(most, count(nk, bound, 1) + 1)
    if m > 0:
        # (the largest logit's equals weigh 1, which is exact)
        least = min(least, int(((w >= m) & ((w >= m + 2.0 ** -42) | (w == 1.0))).sum()))
        most = min(most, int((w >= m - 2.0 ** -42).sum()) if m <= 1 else 1)
    least, most = max(least, 1), max(most, 1)
    first = min(count(least, u * c[least - 1], -1), least - 1) if u > 0 else 0
    last = min(count(most, u * c[most - 1], 1), most - 1) if u > 0 else 0
    return order, w, c, least, most, first, last


def assert_in_range(x, how, token, prob, what=""):
    """One row of float64 logits; returns how many places it may have come to."""
    order, w, c, least, most, first, last = place_range(x, **how)
    V = len(x)
    assert 0 <= token < V, (what, token)
    rank = int(np.flatnonzero(order == token)[0])
    assert first <= rank <= last, (what, how, f"place {rank}, not {first}..{last}")
    near = 2.0 ** -23 * w[rank] / c[least - 1] + (V + 1) * 2.0 ** -41
    assert w[rank] / c[most - 1] - near <= prob <= w[rank] / c[least - 1] + near, (what, how, prob)
    return last - first + 1
