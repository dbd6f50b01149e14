"""GPU parity of attention with capped scores, a bias by distance, windows,
documents and prefixes, over pages and over packed prompts, against float64 within
the bound derived in scored_cases.py."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from paged_cases import NP, PAIRS, Batch, default_scale, to_type, values
from scored_cases import assert_within, scored_rows, seen_by

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged(mlk):
    return importlib.import_module(mlk.__name__ + ".paged")


class Masks:
    """Score functions and masks of a batch, on the host."""

    def __init__(self, batch, H, cap=0.0, bias=False, window=0, prefix=None, docs=None, seed=0):
        rng = np.random.default_rng(seed)
        self.cap, self.window = cap, window
        self.slopes = np.exp2(-8.0 * np.arange(1, H + 1) / H).astype(np.float32) if bias else None
        self.prefix = None
        if prefix is not None:  # "random", or a length for all
            self.prefix = np.array([rng.integers(0, m + 4) if prefix == "random" else prefix
                                    for m in batch.lens], np.int32)
        self.first = None
        if docs is not None:  # "random": documents of up to docs positions; "past": some see nothing
            self.first = np.zeros(batch.T, np.int32)
            for t, s, p in batch.rows():
                d = max(1, batch.lens[s] // 3)
                self.first[t] = p // d * d
                if docs == "past" and t % 3 == 1:
                    self.first[t] = p + 1 if self.prefix is None else 2 ** 31 - 1
                if docs == "negative":
                    self.first[t] = -5
        self.batch = batch

    def handle(self, mlk, paged):
        up = lambda a: None if a is None else mlk.DeviceBuffer.from_array(a)  # noqa: E731
        return paged.Scores(softcap=self.cap, slopes=up(self.slopes), window=self.window,
                            prefix_len=up(self.prefix), first=up(self.first))

    def see(self, t, s, p):
        return seen_by(p, self.batch.lens[s], self.window,
                       None if self.prefix is None else int(self.prefix[s]),
                       None if self.first is None else int(self.first[t]))


class Pages:
    """K and V of a batch's sequences on their pages, NaN elsewhere."""

    def __init__(self, mlk, paged, batch, KV, hd, t, rng, gap=0):
        self.batch, self.t = batch, t
        row = batch.page * KV * hd
        self.kv, host = [], []
        for _ in range(2):
            a = np.full((batch.n_pages, row + gap), np.nan, np.float32)
            view = a[:, :row].reshape(batch.n_pages, batch.page, KV, hd)
            for s, n in enumerate(batch.lens):
                pg, r = batch.slots(s, n)
                view[pg, r] = rng.standard_normal((n, KV, hd))
            host.append(to_type(a, t))
        self.host, self.shape = host, (batch.n_pages, batch.page, KV, hd)
        self.row, self.gap = row, gap
        self.upload(mlk, paged)

    def upload(self, mlk, paged):
        self.bufs = [mlk.DeviceBuffer.from_array(a) for a in self.host]
        n, page, KV, hd = self.shape
        self.handle = paged.PagedCache(*self.bufs, self.t, n, page, KV, hd,
                                       page_stride=self.row + self.gap)

    def view(self, i):
        return self.host[i][:, :self.row].reshape(self.shape)

    def of(self, s):
        pg, r = self.batch.slots(s, self.batch.lens[s])
        return [values(self.view(i)[pg, r], self.t).astype(np.float64) for i in range(2)]


def run_paged(mlk, paged, batch, pages, masks, q, H, act, scale=None, workspace=True, q_stride=None,
              stream=None, dev=None, max_new=None, max_len=None):
    hd = pages.shape[3]
    dev = dev or batch.device(mlk, paged, max_new, max_len)
    dq = mlk.DeviceBuffer.from_array(q)
    out = mlk.DeviceBuffer.from_array(np.full((batch.T, H, hd), 7, NP[act]))
    scores = masks.handle(mlk, paged)
    need = paged.attention_scored_workspace_bytes(pages.handle, dev, scores, H)
    ws = mlk.DeviceBuffer(max(need, 16), np.uint8) if workspace else None
    err = mlk.DeviceBuffer.from_array(np.zeros(1, np.int32))
    paged.attention_scored(pages.handle, dev, scores, dq, out, H, act, scale=scale,
                           q_row_stride=q_stride, workspace=ws, err=err, stream=stream)
    mlk.synchronize()
    assert err.download()[0] == 0
    return out.download()


def check(batch, kv_of, masks, q, got, H, hd, act, scale=None, rows=None):
    scale = scale or default_scale(hd)
    q64 = values(q, act).astype(np.float64).reshape(batch.T, -1)[:, :H * hd].reshape(-1, H, hd)
    raw, got = got, values(got, act)
    kv, written = {}, np.zeros(batch.T, bool)
    for t, s, p in batch.rows():
        written[t] = True
        if rows is not None and t not in rows:
            continue
        if s not in kv:
            kv[s] = kv_of(s)
        out, bound = scored_rows(q64[t], *kv[s], scale, p, masks.see(t, s, p), masks.cap,
                                 masks.slopes, act)
        assert_within(got[t], out, bound, f"token {t} (sequence {s}, position {p})")
    assert (raw[~written] == 7).all(), "rows behind the last sequence were written"


def some_rows(rng, batch, H, most=12):
    n = sum(batch.counts)
    return None if H * n < 600 else set(rng.integers(0, n, most)) | {0, n - 1}


KINDS = {
    "plain": dict(), "cap": dict(cap=20.0), "bias": dict(bias=True), "window": dict(window=50),
    "window 1": dict(window=1), "prefix": dict(prefix="random"), "docs": dict(docs="random"),
    "nothing seen": dict(docs="past"), "cap and bias": dict(cap=5.0, bias=True),
    "window and prefix": dict(window=33, prefix="random", cap=30.0),
    "all": dict(cap=15.0, bias=True, window=70, prefix="random", docs="random"),
    "prefix and nothing": dict(prefix=20, docs="past"), "negative first": dict(docs="negative"),
    "wide window": dict(window=2 ** 40), "whole prefix": dict(prefix=2 ** 31 - 1),
    "negative prefix": dict(prefix=-9),
}
BATCHES = {  # new tokens, lengths, page size, spare rows
    "decode": ([1, 1, 1, 1], [1, 65, 130, 33], 16, 0),
    "decode long": ([1, 1], [1500, 700], 64, 1),
    "chunks": ([5, 17, 0, 1, 130], [5, 100, 40, 33, 130], 16, 3),
    "chunk": ([75], [333], 1, 0),
    "page 512": ([3, 40], [700, 40], 512, 2),
}


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("name", list(BATCHES))
def test_paged(mlk, paged, name, kind, act, ct):
    H, KV, hd = [(32, 8, 128), (8, 2, 64), (6, 2, 80)][len(kind) % 3]
    counts, lens, page, spare = BATCHES[name]
    rng = np.random.default_rng(len(kind) + 7 * len(name))
    batch = Batch(counts, lens, page, spare, seed=H + hd)
    pages = Pages(mlk, paged, batch, KV, hd, ct, rng)
    masks = Masks(batch, H, **KINDS[kind])
    q = to_type(rng.standard_normal((batch.T, H, hd)) * 2, act)
    got = run_paged(mlk, paged, batch, pages, masks, q, H, act)
    check(batch, pages.of, masks, q, got, H, hd, act, rows=some_rows(rng, batch, H))


HEADS = [(4, 2, 16), (8, 1, 256), (12, 12, 64), (71, 1, 64), (5, 5, 33), (16, 2, 96), (64, 8, 128),
         (3, 3, 1), (8, 4, 200)]


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("kind", ["all", "window", "nothing seen"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_paged_heads(mlk, paged, heads, kind, act, ct):
    H, KV, hd = heads
    rng = np.random.default_rng(H + hd)
    batch = Batch([1, 40, 3, 0, 1], [600, 90, 77, 5, 1], 16, 2)
    pages = Pages(mlk, paged, batch, KV, hd, ct, rng)
    masks = Masks(batch, H, **KINDS[kind])
    q = to_type(rng.standard_normal((batch.T, H, hd)) * 2, act)
    got = run_paged(mlk, paged, batch, pages, masks, q, H, act)
    check(batch, pages.of, masks, q, got, H, hd, act, rows=some_rows(rng, batch, H))


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("kind", ["cap", "window", "bias", "all", "nothing seen", "docs"])
def test_paged_long(mlk, paged, kind, act, ct):
    """Positions split over workgroups, with and without a workspace, odd strides,
    gaps between pages, a scale of its own; decode, chunks and both."""
    H, KV, hd = 8, 2, 128 if kind != "all" else 64
    rng = np.random.default_rng(3)
    for counts, lens, page in (([1], [9001], 64), ([1, 1, 1], [5000, 300, 8191], 16),
                               ([300], [5300], 16), ([1, 150, 1], [4000, 3001, 700], 32)):
        batch = Batch(counts, lens, page, 1)
        for gap, extra, ws in ((0, 0, True), (3, 5, False)):
            pages = Pages(mlk, paged, batch, KV, hd, ct, rng, gap=gap)
            masks = Masks(batch, H, **dict(KINDS[kind], **(dict(window=1000) if kind == "window" else {})))
            q = to_type(rng.standard_normal((batch.T, H * hd + extra)), act)
            got = run_paged(mlk, paged, batch, pages, masks, q, H, act, scale=0.15, workspace=ws,
                            q_stride=H * hd + extra)
            check(batch, pages.of, masks, q, got, H, hd, act, scale=float(np.float32(0.15)),
                  rows=set(rng.integers(0, sum(counts), 5)) | {0, sum(counts) - 1})


@pytest.mark.parametrize("act,ct", PAIRS)
def test_bounds_far_above_what_comes(mlk, paged, act, ct):
    """The host's bounds (new tokens, lengths) twenty times what the device finds."""
    H, KV, hd = 8, 2, 64
    rng = np.random.default_rng(4)
    batch = Batch([1, 2, 30, 1], [40, 99, 60, 300], 16, 60)
    batch.table = np.pad(batch.table, ((0, 0), (0, 400)), constant_values=-1)
    batch.width = batch.table.shape[1]
    pages = Pages(mlk, paged, batch, KV, hd, ct, rng)
    for kind in ("all", "window", "bias"):
        masks = Masks(batch, H, **KINDS[kind])
        q = to_type(rng.standard_normal((batch.T, H, hd)), act)
        got = run_paged(mlk, paged, batch, pages, masks, q, H, act, max_new=90, max_len=6000)
        check(batch, pages.of, masks, q, got, H, hd, act)


def test_many_sequences(mlk, paged):
    """More sequences than workers, windows shorter and longer than they are."""
    H, KV, hd = 8, 2, 64
    rng = np.random.default_rng(14)
    n = 1500
    counts = [int(c) for c in rng.integers(0, 3, n)]
    lens = [int(max(c, m)) for c, m in zip(counts, rng.integers(1, 700, n))]
    batch = Batch(counts, lens, 32)
    pages = Pages(mlk, paged, batch, KV, hd, "bf16", rng)
    q = to_type(rng.standard_normal((batch.T, H, hd)), "bf16")
    for kw in (dict(window=64, cap=10.0), dict(bias=True, docs="random"), dict(window=3000)):
        masks = Masks(batch, H, **kw)
        got = run_paged(mlk, paged, batch, pages, masks, q, H, "bf16")
        check(batch, pages.of, masks, q, got, H, hd, "bf16", rows=set(rng.integers(0, batch.T, 60)))


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("ones", [7, 600])
def test_chunks_beside_single_tokens(mlk, paged, ones, act, ct):
    """Both kinds of rows with parts to join, in batches of fewer and of more sequences than
    workers; the plain entry over the same ones."""
    H, KV, hd = 8, 2, 64
    rng = np.random.default_rng(15)
    counts = [1] * ones + [130] + [1] * ones
    lens = [int(n) for n in rng.integers(600 if ones == 7 else 1, 2000 if ones == 7 else 700, 2 * ones + 1)]
    lens[ones] = 1900
    batch = Batch(counts, lens, 32)
    pages = Pages(mlk, paged, batch, KV, hd, ct, rng)
    q = to_type(rng.standard_normal((batch.T, H, hd)), act)
    rows = set(rng.integers(0, batch.T, 20)) | {ones, ones + 64, ones + 129}
    for kw in (dict(window=1000, cap=10.0), dict(bias=True, prefix="random")):
        masks = Masks(batch, H, **kw)
        got = run_paged(mlk, paged, batch, pages, masks, q, H, act)
        check(batch, pages.of, masks, q, got, H, hd, act, rows=rows)
    dev = batch.device(mlk, paged)
    out = mlk.DeviceBuffer.from_array(np.full((batch.T, H, hd), 7, NP[act]))
    ws = mlk.DeviceBuffer(max(paged.attention_workspace_bytes(pages.handle, dev, H, act), 16), np.uint8)
    paged.attention(pages.handle, dev, mlk.DeviceBuffer.from_array(q), out, H, act, workspace=ws)
    mlk.synchronize()
    check(batch, pages.of, Masks(batch, H), q, out.download(), H, hd, act, rows=rows)


class FarPages(Pages):
    """Pages 2^29 elements apart."""

    def upload(self, mlk, paged):
        n, page, KV, hd = self.shape
        stride, size = 1 << 29, self.host[0].itemsize
        self.bufs = [mlk.DeviceBuffer(((n - 1) * stride + self.row) * size, np.uint8) for _ in range(2)]
        for buf, a in zip(self.bufs, self.host):
            for i in range(n):
                one = np.ascontiguousarray(a[i, :self.row])
                mlk.check(mlk.lib.mlk_memcpy(buf.offset(i * stride * size), one.ctypes.data, one.nbytes, mlk.H2D))
        self.handle = paged.PagedCache(*self.bufs, self.t, n, page, KV, hd, page_stride=stride)


@pytest.mark.parametrize("counts,lens", [([1, 2], [700, 300]), ([70, 1], [400, 650])])
def test_offsets_past_32_bits(mlk, paged, counts, lens):
    H, KV, hd = 8, 2, 128
    rng = np.random.default_rng(16)
    batch = Batch(counts, lens, 64)
    pages = FarPages(mlk, paged, batch, KV, hd, "bf16", rng)
    assert batch.n_pages > 8 and batch.table.max() >= 8
    q = to_type(rng.standard_normal((batch.T, H, hd)), "bf16")
    for kw in (dict(cap=10.0, window=250), dict(bias=True)):
        masks = Masks(batch, H, **kw)
        got = run_paged(mlk, paged, batch, pages, masks, q, H, "bf16")
        check(batch, pages.of, masks, q, got, H, hd, "bf16", rows=some_rows(rng, batch, H))


# ------------------------------------------------------------------ packed

def run_packed(mlk, paged, batch, masks, q, k, v, H, KV, hd, act, strides=(None,) * 3,
               workspace=True, offset=(0, 0, 0)):
    size = np.dtype(NP[act]).itemsize
    bufs = [mlk.DeviceBuffer.from_array(a) for a in (q, k, v)]
    start = mlk.DeviceBuffer.from_array(batch.start)
    out = mlk.DeviceBuffer.from_array(np.full((batch.T, H, hd), 7, NP[act]))
    most = max(max(batch.counts), 1)
    scores = masks.handle(mlk, paged)
    need = paged.attention_packed_scored_workspace_bytes(scores, len(batch.counts), batch.T, most,
                                                         H, KV, hd)
    ws = mlk.DeviceBuffer(max(need, 16), np.uint8) if workspace else None
    err = mlk.DeviceBuffer.from_array(np.zeros(1, np.int32))
    ptr = [b.offset(o * size) for b, o in zip(bufs, offset)]
    paged.attention_packed_scored(act, scores, *ptr, start, len(batch.counts), batch.T, most, H, KV,
                                  hd, out, q_row_stride=strides[0], k_row_stride=strides[1],
                                  v_row_stride=strides[2], workspace=ws, err=err)
    mlk.synchronize()
    assert err.download()[0] == 0
    return out.download()


def packed_kv(batch, k, v, act):
    k, v = (values(a, act).astype(np.float64) for a in (k, v))
    return lambda s: (k[batch.start[s]:batch.start[s + 1]], v[batch.start[s]:batch.start[s + 1]])


PACKED = {
    "one": ([1], 0), "empty among": ([0, 3, 0, 0, 64, 1, 0], 2), "ragged": ([33, 1, 129, 200, 63], 1),
    "long": ([700], 0), "many": ([1] * 70 + [5] * 70, 0), "all empty": ([0, 0], 4),
}


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("name", list(PACKED))
def test_packed(mlk, paged, name, kind, act):
    H, KV, hd = [(32, 8, 128), (8, 2, 64), (8, 1, 256), (6, 2, 80)][len(kind) % 4]
    counts, spare = PACKED[name]
    rng = np.random.default_rng(H * hd)
    batch = Batch(counts, None, spare=spare)
    qkv = [to_type(rng.standard_normal((batch.T, n, hd)), act) for n in (H, KV, KV)]
    for a in qkv:  # what lies behind the last sequence is not read
        a[sum(counts):] = to_type(np.float32([np.nan]), act)[0]
    masks = Masks(batch, H, **KINDS[kind])
    got = run_packed(mlk, paged, batch, masks, *qkv, H, KV, hd, act)
    check(batch, packed_kv(batch, qkv[1], qkv[2], act), masks, qkv[0], got, H, hd, act,
          rows=None if not sum(counts) else some_rows(rng, batch, H))


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["cap", "docs", "prefix", "window", "all"])
def test_packed_long_over_a_fused_projection(mlk, paged, act, kind):
    H, KV, hd = 8, 2, 128
    batch = Batch([1900, 3, 700], None, spare=1)
    rng = np.random.default_rng(4)
    for pad, ws in ((0, True), (1, False)):
        width = (H + 2 * KV) * hd + pad
        qkv = to_type(rng.standard_normal((batch.T, width)), act)
        masks = Masks(batch, H, **KINDS[kind])
        got = run_packed(mlk, paged, batch, masks, qkv, qkv, qkv, H, KV, hd, act,
                         strides=(width,) * 3, offset=(0, H * hd, (H + KV) * hd), workspace=ws)
        parts = np.split(qkv[:, :(H + 2 * KV) * hd], [H * hd, (H + KV) * hd], axis=1)
        q, k, v = (p.reshape(batch.T, -1, hd) for p in parts)
        check(batch, packed_kv(batch, k, v, act), masks, q, got, H, hd, act,
              rows=set(rng.integers(0, 2603, 10)) | {0, 1899, 1900, 2602})


# ------------------------------------------------------------------ what must not reach a result

@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("hd,n", [(128, 70), (64, 6), (24, 6), (256, 35)])
def test_unseen_positions_do_not_reach_a_token(mlk, paged, act, ct, value, hd, n):
    """Non-finite K and V where some tokens do not see them, by window, document or
    order: those tokens as without them, the others non-finite."""
    H, KV = 4, 2
    rng = np.random.default_rng(5)
    batch = Batch([n, 1], [n + 90, 50], 16)
    for kw in (dict(window=40), dict(docs="random", cap=9.0), dict(prefix=n + 40, bias=True)):
        pages = Pages(mlk, paged, batch, KV, hd, ct, rng)
        masks = Masks(batch, H, **kw)
        q = to_type(rng.standard_normal((batch.T, H, hd)), act)
        good = [a.copy() for a in pages.host]
        for pos in (60, 90 + n // 2):
            pg, r = batch.slots(0, n + 90)
            for which in (0, 1):
                pages.host = [a.copy() for a in good]
                pages.view(which)[pg[pos], r[pos], 1] = to_type(np.float32([value]), ct)[0]
                pages.upload(mlk, paged)
                got = run_paged(mlk, paged, batch, pages, masks, q, H, act)
                sees = np.array([masks.see(t, s, p)[pos] if s == 0 else False
                                 for t, s, p in batch.rows()])
                clean = pages.host
                pages.host = good
                check(batch, pages.of, masks, q, got, H, hd, act,
                      rows=set(np.flatnonzero(~sees)[-12:]) | set(np.flatnonzero(~sees)[:3]))
                pages.host = clean
                g = values(got, act).reshape(batch.T, KV, H // KV, hd)
                assert np.isfinite(g[~sees]).all() and np.isfinite(g[:, 0]).all()
                if which == 1:
                    assert not np.isfinite(g[sees][:, 1]).any()
                elif np.isnan(value):
                    assert np.isnan(g[sees][:, 1]).all()


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("n", [3, 400])
def test_non_finite_values_far_apart(mlk, paged, act, ct, n):
    """V infinite at positions thousands apart, in tiles that tokens of one document see
    and those of the next do not: each token gets what it sees, sum and sign."""
    H, KV, hd, m = 4, 2, 64, 3500
    rng = np.random.default_rng(21)
    batch = Batch([n, 1], [m, 900], 16)
    pages = Pages(mlk, paged, batch, KV, hd, ct, rng)
    masks = Masks(batch, H, cap=20.0)
    masks.first = np.zeros(batch.T, np.int32)
    masks.first[n // 2:n] = 2900  # the second half of the new tokens: a document of their own
    places = {(5, 0): np.inf, (1700, 1): -np.inf, (2890, 2): np.inf, (2950, 3): np.inf, (10, 4): np.inf,
              (2000, 4): -np.inf, (m - 2, 5): -np.inf}
    view = pages.view(1)
    for (pos, d), x in places.items():
        pg, r = batch.slots(0, m)
        view[pg[pos], r[pos], 0, d] = to_type(np.float32([x]), ct)[0]
    pages.upload(mlk, paged)
    q = to_type(rng.standard_normal((batch.T, H, hd)), act)
    got = values(run_paged(mlk, paged, batch, pages, masks, q, H, act), act).reshape(batch.T, KV, H // KV, hd)
    for t, s, p in batch.rows():
        see = masks.see(t, s, p)
        bad = {}
        for (pos, d), x in places.items():
            if s == 0 and pos < len(see) and see[pos]:
                bad.setdefault(d, set()).add(x)
        for d in range(hd):
            g = got[t, 0, :, d]
            if d not in bad:
                assert np.isfinite(g).all(), (t, d)
            elif len(bad[d]) > 1:
                assert np.isnan(g).all(), (t, d)
            elif act != "f32":
                assert (g == next(iter(bad[d]))).all(), (t, d)
            else:  # fp32's pieces may meet it as inf - inf
                assert not np.isfinite(g).any(), (t, d)
        assert np.isfinite(got[t, 1]).all()


@pytest.mark.parametrize("act,ct", PAIRS)
def test_large_scores_are_capped(mlk, paged, act, ct):
    """Scores hundreds of times the cap, of either sign: tanh at its ends."""
    H, KV, hd = 4, 2, 64
    rng = np.random.default_rng(9)
    batch = Batch([1, 40], [300, 190], 16)
    for cap, size in ((1.0, 40.0), (50.0, 200.0), (1e-3, 1.0), (1e4, 3.0)):
        pages = Pages(mlk, paged, batch, KV, hd, ct, rng)
        masks = Masks(batch, H, cap=cap)
        q = to_type(rng.standard_normal((batch.T, H, hd)) * size, act)
        got = run_paged(mlk, paged, batch, pages, masks, q, H, act)
        check(batch, pages.of, masks, q, got, H, hd, act, rows=set(range(0, batch.T, 6)))


def test_scored_without_functions_is_the_plain_call(mlk, paged):
    """No cap, bias or mask: the plain entry's result, within both bounds."""
    H, KV, hd = 8, 2, 128
    rng = np.random.default_rng(10)
    batch = Batch([1, 60, 1], [700, 90, 33], 16)
    for act, ct in PAIRS:
        pages = Pages(mlk, paged, batch, KV, hd, ct, rng)
        masks = Masks(batch, H)
        q = to_type(rng.standard_normal((batch.T, H, hd)), act)
        got = run_paged(mlk, paged, batch, pages, masks, q, H, act)
        check(batch, pages.of, masks, q, got, H, hd, act, rows=set(range(0, 62, 5)))


def test_sequences_out_of_bounds_are_left_alone(mlk, paged):
    """A sequence longer than the bound, one with more new tokens than its length,
    a page outside the cache: raised, the others as they should be."""
    H, KV, hd = 8, 2, 64
    rng = np.random.default_rng(11)
    batch = Batch([1, 2, 3, 1], [90, 60, 70, 44], 16)
    pages = Pages(mlk, paged, batch, KV, hd, "f16", rng)
    masks = Masks(batch, H, cap=20.0, window=50, prefix="random", docs="random")
    q = to_type(rng.standard_normal((batch.T, H, hd)), "f32")
    for wrong in ("len", "count", "page"):
        lens, table = np.asarray(batch.lens, np.int32), batch.table.copy()
        if wrong == "len":
            lens[1] = 5000
        elif wrong == "count":
            lens[1] = 1
        else:
            table[1, 3] = batch.n_pages
        keep = [mlk.DeviceBuffer.from_array(a) for a in (batch.start, lens, table)]
        dev = paged.PagedBatch(*keep, 4, batch.T, batch.width, 3, 90)
        out = mlk.DeviceBuffer.from_array(np.full((batch.T, H, hd), 7, np.float32))
        err = mlk.DeviceBuffer.from_array(np.zeros(1, np.int32))
        paged.attention_scored(pages.handle, dev, masks.handle(mlk, paged),
                               mlk.DeviceBuffer.from_array(q), out, H, "f32", err=err)
        mlk.synchronize()
        assert err.download()[0] != 0
        got = out.download()
        if wrong != "page":
            assert (got[1:3] == 7).all()
            got[1:3] = run_paged(mlk, paged, batch, pages, masks, q, H, "f32")[1:3]
        check(batch, pages.of, masks, q, got, H, hd, "f32", rows={0, 3, 4, 5, 6})


@pytest.mark.parametrize("act,ct", [("f32", "f16"), ("bf16", "bf16")])
def test_replays_over_growing_sequences(mlk, paged, act, ct):
    """A captured call replayed with other lengths and prefixes within its bounds."""
    H, KV, hd = 8, 2, 128
    rng = np.random.default_rng(12)
    stream = mlk.Stream()
    big = Batch([1, 1, 40], [3000, 900, 500], 16)
    pages = Pages(mlk, paged, big, KV, hd, ct, rng)
    masks = Masks(big, H, cap=30.0, window=700, prefix="random", bias=True)
    q = to_type(rng.standard_normal((big.T, H, hd)), act)
    up = mlk.DeviceBuffer.from_array
    dq, out = up(q), up(np.zeros((big.T, H, hd), NP[act]))
    dev = big.device(mlk, paged)
    scores = masks.handle(mlk, paged)
    ws = mlk.DeviceBuffer(max(paged.attention_scored_workspace_bytes(pages.handle, dev, scores, H), 16), np.uint8)

    def call(to, s):
        paged.attention_scored(pages.handle, dev, scores, dq, to, H, act, workspace=ws, stream=s)

    call(out, stream.handle)
    stream.synchronize()
    with mlk.Graph.capture(stream) as g:
        call(out, stream.handle)
    for lens in ([3000, 900, 500], [1, 2, 40], [2900, 33, 64], [17, 880, 499]):
        big.lens = lens
        big.keep[1].upload(np.asarray(lens, np.int32))
        masks.prefix[:] = rng.integers(0, 60, 3)
        scores._keep[1].upload(masks.prefix)
        g.launch()
        stream.synchronize()
        got = out.download()
        check(big, pages.of, masks, q, got, H, hd, act, rows={0, 1, 2, 20, 41})
        eager = up(np.zeros((big.T, H, hd), NP[act]))
        call(eager, None)
        mlk.synchronize()
        np.testing.assert_array_equal(got.view(np.uint8), eager.download().view(np.uint8))
