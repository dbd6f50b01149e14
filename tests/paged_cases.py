"""Helpers of the paged-cache and packed attention tests: element types in
numpy, ragged batches on the host, float64 results and their error bounds.

attention_bound, for output element (h, d) of a token over n positions, u =
2^-24, pav = sum_j w_j |v_jd|:
  - a score is a sum of hd products, each within 2^-20 (16 u) of itself or, for
    an element of q more than 2^17 below its row's largest, within 2^-38 of that
    largest one times |k|; the fp32 sum adds gamma_{hd+2}, the scale (times
    log2 e, rounded) 3 u: D = (gamma_{hd+2} + 19 u) scale sum |q k| + 2^-38 scale
    max|q| sum |k|, and a score error D moves w_j by 2 D relatively;
  - exp: the argument (at most 32 where w_j matters) is rounded once, 32 u, and
    the instruction is good to 2 u; the sum of n terms and the division add
    (n + 4) u, the products' pieces 16 u, and 2^-38 sum |v_j| where w_j is more
    than 2^17 below the largest: (n + 54) u in all;
  - 16-bit activations: w_j is rounded to the type (e = eps / 2 of itself;
    fp16 below its normal range, of values scaled by 2^14, 2^-39 absolutely) and
    so is the output (e |out| + the type's smallest half step).
"""
from __future__ import annotations

import math

import numpy as np

U = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}
NP = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


def to_type(x, t):
    """fp32 values rounded to type t (bf16 as its bits)."""
    x = np.ascontiguousarray(x, np.float32)
    if t != "bf16":
        return x.astype(NP[t])
    b = x.view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def values(a, t):
    """Elements of type t as float32."""
    if t != "bf16":
        return np.asarray(a, np.float32)
    return (np.asarray(a, np.uint32) << 16).view(np.float32)


class Batch:
    """New tokens (counts) of sequences of the given lengths (None: packed),
    pages scattered over the cache, `spare` token rows behind the last."""

    def __init__(self, counts, lens, page=16, spare=0, seed=0, extra_pages=3):
        self.counts = list(counts)
        self.lens = list(lens if lens is not None else counts)
        self.start = np.concatenate([[0], np.cumsum(self.counts)]).astype(np.int32)
        self.T = int(self.start[-1]) + spare
        self.page = page
        used = [-(-n // page) for n in self.lens]
        self.n_pages = sum(used) + extra_pages
        self.width = max(max(used), 1)
        order = np.random.default_rng(seed).permutation(self.n_pages)
        self.table = np.full((len(used), self.width), -1, np.int32)  # unused entries: no page
        at = 0
        for s, n in enumerate(used):
            self.table[s, :n] = order[at:at + n]
            at += n

    def rows(self):
        """(token row, sequence, position) of every token."""
        for s, (n, m) in enumerate(zip(self.counts, self.lens)):
            for i in range(n):
                yield int(self.start[s]) + i, s, m - n + i

    def slots(self, s, n):
        """(page, row) of positions 0 .. n - 1 of sequence s."""
        j = np.arange(n)
        return self.table[s, j // self.page], j % self.page

    def device(self, mlk, paged, max_new=None, max_len=None):
        self.keep = [mlk.DeviceBuffer.from_array(a) for a in
                     (self.start, np.asarray(self.lens, np.int32), self.table)]
        return paged.PagedBatch(*self.keep, len(self.counts), self.T, self.width,
                                max_new or max(max(self.counts), 1), max_len or max(self.lens))


def exact_rows(q, k, v, scale):
    """q [H, hd], k and v [n, KV, hd] (float64): out, pav [H, hd] and the score
    bound D of one token over all n positions."""
    H, hd = q.shape
    g = H // k.shape[1]
    out, pav = np.empty((H, hd)), np.empty((H, hd))
    gamma = (hd + 2) * U / (1 - (hd + 2) * U) + 19 * U
    d = 0.0
    for h in range(H):
        kk, vv = k[:, h // g], v[:, h // g]
        s = kk @ q[h] * scale
        w = np.exp(s - s.max())
        w /= w.sum()
        out[h], pav[h] = w @ vv, w @ np.abs(vv)
        d = max(d, gamma * scale * float((np.abs(kk) @ np.abs(q[h])).max()) + 2.0 ** -38 * scale
                * float(np.abs(q[h]).max() * np.abs(kk).sum(1).max()))
    return out, pav, d


def assert_close(got, out, pav, d, n, vsum, t, what):
    e = 0.0 if t == "f32" else HALF_STEP[t]
    bound = (2 * d + (n + 54) * U + e) * pav * (1 + 2 * d) + 2.0 ** -38 * vsum
    bound = bound + HALF_STEP[t] * (np.abs(out) + bound) + TINY[t] + 1e-30
    err = np.abs(np.asarray(got, np.float64) - out)
    bad = ~(err <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {err.size} beyond the bound; worst err "
                           f"{float(np.nanmax(err)):.3e}, its bound "
                           f"{float(bound.flat[np.nanargmax(err)]):.3e}")


def default_scale(hd):
    return float(np.float32(1.0 / math.sqrt(hd)))
