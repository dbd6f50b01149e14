"""Float64 results and error bounds of attention with score functions and masks.

For output element (h, d) of a token, u = 2^-24, over the positions it sees (w_j
their weights, x_j the scores after cap and bias):
  - D_j, the error of x_j: scale q . k_j as paged_cases.py derives it ((gamma_{hd+2}
    + 19 u) scale sum |q k| + 2^-38 scale max|q| sum |k|); the cap does not widen it
    (its slope is at most 1) and adds 16 u cap (two products, the division by cap
    and tanh to within 8 u); the bias and its difference add 6 u (slope |p - j| + |x_j|);
  - the weight of j moves by D_j + sum_i w_i D_i relatively, to first order; twice
    that covers the rest while it is below 1/2;
  - exp, sums, division, the weights' pieces and the output's rounding as there:
    (n + 54) u, 2^-38 sum |v_j|, and for 16-bit activations the type's half step of
    w_j and of the result.
"""
from __future__ import annotations

import numpy as np

from paged_cases import HALF_STEP, TINY, U


def seen_by(p, m, window=0, prefix=None, first=None):
    """The positions of 0 .. m - 1 that the token at position p sees, by the definition."""
    j = np.arange(m)
    see = j <= p
    if prefix is not None:
        see |= (j < prefix) & (p < prefix)
    if window:
        see &= j > p - window
    if first is not None:
        see &= j >= first
    return see


def scored_rows(q, k, v, scale, p, see, cap=0.0, slopes=None, type="f32"):
    """q [H, hd] at position p over the positions `see` of k, v [n, KV, hd], float64:
    out [H, hd] and its bound."""
    H, hd = q.shape
    g = H // k.shape[1]
    if not see.any():
        return np.zeros((H, hd)), np.zeros((H, hd))
    j = np.flatnonzero(see)
    gamma = (hd + 2) * U / (1 - (hd + 2) * U) + 19 * U
    e = 0.0 if type == "f32" else HALF_STEP[type]
    out, bound = np.empty((H, hd)), np.empty((H, hd))
    for h in range(H):
        kk, vv = k[j, h // g], v[j, h // g]
        x = kk @ q[h] * scale
        D = gamma * scale * (np.abs(kk) @ np.abs(q[h])) + \
            2.0 ** -38 * scale * np.abs(q[h]).max() * np.abs(kk).sum(1)
        if cap:
            x = cap * np.tanh(x / cap)
            D = D + 16 * U * cap
        if slopes is not None:
            b = float(slopes[h]) * np.abs(p - j)
            D = D + 6 * U * (b + np.abs(x))
            x = x - b
        w = np.exp(x - x.max())
        w /= w.sum()
        out[h] = w @ vv
        pav = w @ np.abs(vv)
        moved = 2 * ((w * D) @ np.abs(vv) + float(w @ D) * pav)
        b = moved + ((len(j) + 54) * U + e) * pav + 2.0 ** -38 * np.abs(vv).sum(0)
        bound[h] = b + HALF_STEP[type] * (np.abs(out[h]) + b) + TINY[type] + 1e-30
    return out, bound


def assert_within(got, out, bound, what):
    err = np.abs(np.asarray(got, np.float64) - out)
    bad = ~(err <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {err.size} beyond the bound; worst err "
                           f"{float(np.nanmax(err)):.3e}, its bound "
                           f"{float(bound.flat[np.nanargmax(err)]):.3e}")
