"""GPU parity of the operators for many sequences: append to a paged KV cache
with RoPE on the way, attention over it, and attention over packed prompts.

The append is bit-exact: what mlk_rope_f32 leaves, rounded to the stored type.
Attention is held to the bound derived in paged_cases.py against float64."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from paged_cases import (NP, PAIRS, Batch, assert_close, default_scale, exact_rows, to_type,
                         values)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged(mlk):
    return importlib.import_module(mlk.__name__ + ".paged")


class Cache:
    """Pages filled with random values, NaN where no position of the batch
    lies; `gap` unused elements between pages."""

    def __init__(self, mlk, paged, batch, KV, hd, t, rng, gap=0, fill=True):
        self.batch, self.KV, self.hd, self.t = batch, KV, hd, t
        row = batch.page * KV * hd
        self.stride = row + gap
        self.host = []
        for _ in range(2):
            a = np.full((batch.n_pages, self.stride), np.nan, np.float32)
            if fill:
                for s, n in enumerate(batch.lens):
                    pg, r = batch.slots(s, n)
                    view = a[:, :row].reshape(batch.n_pages, batch.page, KV, hd)
                    view[pg, r] = rng.standard_normal((n, KV, hd))
            self.host.append(to_type(a, t))
        self.upload(mlk)
        self.handle = paged.PagedCache(self.k, self.v, t, batch.n_pages, batch.page, KV, hd,
                                       page_stride=self.stride)

    def upload(self, mlk):
        self.k, self.v = (mlk.DeviceBuffer.from_array(a) for a in self.host)

    def pages(self, which, src=None):
        """[n_pages, page, KV, hd] view of the host copy (or of src)."""
        a = self.host[which] if src is None else src
        n = self.batch.page * self.KV * self.hd
        return a[:, :n].reshape(self.batch.n_pages, self.batch.page, self.KV, self.hd)

    def gathered(self, s, n):
        """Positions 0 .. n - 1 of sequence s as float64 k, v [n, KV, hd]."""
        pg, r = self.batch.slots(s, n)
        return [values(self.pages(i)[pg, r], self.t).astype(np.float64) for i in range(2)]


def run_paged(mlk, paged, batch, cache, q, H, act, scale=None, workspace=True, q_stride=None,
              stream=None, dev=None):
    """out [T, H, hd] in type act (rows nobody writes hold a marker)."""
    hd = cache.hd
    dev = dev or batch.device(mlk, paged)
    dq = mlk.DeviceBuffer.from_array(q)
    marker = np.full((batch.T, H, hd), 7, NP[act])
    out = mlk.DeviceBuffer.from_array(marker)
    need = paged.attention_workspace_bytes(cache.handle, dev, H, act)
    ws = mlk.DeviceBuffer(max(need, 16), np.uint8) if workspace else None
    err = mlk.DeviceBuffer.from_array(np.zeros(1, np.int32))
    paged.attention(cache.handle, dev, dq, out, H, act, scale=scale, q_row_stride=q_stride,
                    workspace=ws, err=err, stream=stream)
    mlk.synchronize()
    assert err.download()[0] == 0
    return out.download()


def check_paged(batch, cache, q, got, H, act, scale=None, rows=None):
    hd = cache.hd
    scale = scale or default_scale(hd)
    q64 = values(q, act).astype(np.float64).reshape(batch.T, -1)[:, :H * hd].reshape(-1, H, hd)
    kv = {}
    written = np.zeros(batch.T, bool)
    for t, s, p in batch.rows():
        written[t] = True
        if rows is not None and t not in rows:
            continue
        if s not in kv:
            kv[s] = cache.gathered(s, batch.lens[s])
        k, v = (a[:p + 1] for a in kv[s])
        out, pav, d = exact_rows(q64[t], k, v, scale)
        vsum = np.repeat(np.abs(v).sum(0), H // cache.KV, axis=0)
        assert_close(values(got[t], act), out, pav, d, p + 1, vsum, act,
                     f"token {t} (sequence {s}, position {p})")
    assert (got[~written] == 7).all(), "rows behind the last sequence were written"


HEADS = [(4, 2, 16), (32, 8, 128), (8, 1, 256), (6, 2, 80), (12, 12, 64), (71, 1, 64), (5, 5, 33),
         (16, 2, 96), (64, 8, 128), (3, 3, 1), (8, 4, 200)]
BATCHES = {  # new tokens, lengths, page size, spare rows
    "one": ([1], [1], 16, 0),
    "decode": ([1, 1, 1, 1], [1, 65, 130, 33], 16, 0),
    "decode long": ([1, 1], [1500, 700], 64, 1),
    "two each": ([2, 2, 2], [2, 64, 77], 8, 0),
    "chunks": ([5, 17, 0, 1, 130], [5, 100, 40, 33, 130], 16, 3),
    "chunk": ([75], [333], 1, 0),
    "page 512": ([3, 40], [700, 40], 512, 2),
}


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("name", list(BATCHES))
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_paged_attention(mlk, paged, heads, name, act, ct):
    H, KV, hd = heads
    counts, lens, page, spare = BATCHES[name]
    rng = np.random.default_rng(hash((H, hd, len(counts))) % 1000)
    batch = Batch(counts, lens, page, spare, seed=H + hd)
    cache = Cache(mlk, paged, batch, KV, hd, ct, rng)
    q = to_type(rng.standard_normal((batch.T, H, hd)), act)
    got = run_paged(mlk, paged, batch, cache, q, H, act)
    some = None if H * batch.T < 800 else set(rng.integers(0, batch.T, 12)) | {0, sum(counts) - 1}
    check_paged(batch, cache, q, got, H, act, rows=some)


@pytest.mark.parametrize("act,ct", PAIRS)
def test_paged_attention_strides_and_no_workspace(mlk, paged, act, ct):
    """q as a slice of a fused projection's odd-strided rows, gaps between
    pages, no workspace, a scale of its own."""
    H, KV, hd = 8, 2, 64
    rng = np.random.default_rng(3)
    batch = Batch([1, 9, 1], [900, 300, 17], 16, 1)
    for gap, stride in ((0, H * hd + 2 * KV * hd), (3, H * hd + 5)):
        cache = Cache(mlk, paged, batch, KV, hd, ct, rng, gap=gap)
        q = to_type(rng.standard_normal((batch.T, stride)), act)
        for ws in (True, False):
            got = run_paged(mlk, paged, batch, cache, q, H, act, scale=0.3, workspace=ws,
                            q_stride=stride)
            check_paged(batch, cache, q, got, H, act, scale=float(np.float32(0.3)))


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("hd", [64, 128, 40])
def test_paged_attention_large_and_small_values(mlk, paged, act, ct, hd):
    """Scores whose softmax is one position, and ones far below fp16's range."""
    H, KV = 4, 2
    rng = np.random.default_rng(9)
    batch = Batch([1, 40], [300, 190], 16)
    for qs, ks in ((30.0, 3.0), (1e-6, 1.0), (1e-3, 1e-3)):
        cache = Cache(mlk, paged, batch, KV, hd, ct, rng)
        cache.host[0] = to_type(values(cache.host[0], ct) * np.float32(ks), ct)
        cache.upload(mlk)
        cache.handle = paged.PagedCache(cache.k, cache.v, ct, batch.n_pages, batch.page, KV, hd)
        x = rng.standard_normal((batch.T, H, hd)) * qs
        x[..., ::3] *= 1e-3
        q = to_type(x, act)
        got = run_paged(mlk, paged, batch, cache, q, H, act)
        check_paged(batch, cache, q, got, H, act, rows=set(range(0, batch.T, 7)) | {batch.T - 1})


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("hd,n", [(128, 70), (64, 6), (24, 6), (256, 35)])
def test_later_tokens_do_not_reach_earlier_ones(mlk, paged, act, ct, value, hd, n):
    """Non-finite K and V at one new token: the tokens before it as without it,
    itself and later ones non-finite where its value enters."""
    H, KV = 4, 2
    rng = np.random.default_rng(5)
    batch = Batch([n, 1], [n + 37, 50], 16)
    cache = Cache(mlk, paged, batch, KV, hd, ct, rng)
    q = to_type(rng.standard_normal((batch.T, H, hd)), act)
    bad = n - 3  # the token whose rows are bad
    pg, r = batch.slots(0, n + 37)
    pos = 37 + bad
    good = [a.copy() for a in cache.host]
    for which, dims in ((1, slice(0, hd)), (0, slice(0, 1)), (1, slice(hd // 2, hd // 2 + 1))):
        cache.host = [a.copy() for a in good]
        cache.pages(which)[pg[pos], r[pos], 1, dims] = to_type(np.float32([value]), ct)[0]
        cache.upload(mlk)
        cache.handle = paged.PagedCache(cache.k, cache.v, ct, batch.n_pages, batch.page, KV, hd)
        got = run_paged(mlk, paged, batch, cache, q, H, act)
        ok = [t for t, s, p in batch.rows() if s == 1 or p < pos]
        check_paged(batch, cache, q, got, H, act, rows=set(ok[-30:]))
        g = values(got, act).reshape(batch.T, KV, H // KV, hd)
        assert np.isfinite(g[:bad]).all() and np.isfinite(g[:, 0]).all()
        assert np.isfinite(g[n:]).all()
        if which == 1:
            assert not np.isfinite(g[bad:n, 1][..., dims]).any()
            other = np.ones(hd, bool)
            other[dims] = False
            assert np.isfinite(g[bad:n, 1][..., other]).all()
            if act != "f32" and not np.isnan(value):  # fp32's pieces meet it as inf - inf
                assert (g[bad:n, 1][..., dims] == value).all()


def test_paged_attention_counts_every_position_once(mlk, paged):
    """Equal scores, values coding their position: the mean of 0 .. p, over
    many chunks of a long context."""
    H, KV, hd = 8, 2, 64
    for act, ct in PAIRS:
        batch = Batch([1, 3, 1], [9001, 5000, 4097], 64)
        cache = Cache(mlk, paged, batch, KV, hd, ct, np.random.default_rng(1))
        for s, n in enumerate(batch.lens):
            pg, r = batch.slots(s, n)
            cache.pages(0)[pg, r] = to_type(np.float32([0.5]), ct)[0]
            ones = np.zeros((n, KV, hd), np.float32)  # dim d: one at positions j % hd == d
            ones[np.arange(n), :, np.arange(n) % hd] = 1
            cache.pages(1)[pg, r] = to_type(ones, ct)
        cache.upload(mlk)
        cache.handle = paged.PagedCache(cache.k, cache.v, ct, batch.n_pages, batch.page, KV, hd)
        q = to_type(np.ones((batch.T, H, hd)), act)
        got = values(run_paged(mlk, paged, batch, cache, q, H, act), act)
        for t, s, p in batch.rows():
            want = np.bincount(np.arange(p + 1) % hd, minlength=hd) / (p + 1)
            tol = 2.0 ** -19 if act == "f32" else 2.0 ** -6 if act == "bf16" else 2.0 ** -9
            assert np.abs(got[t] / want - 1).max() <= tol, (act, ct, t)


# ------------------------------------------------------------------ packed

def run_packed(mlk, paged, batch, q, k, v, H, KV, hd, act, strides=(None,) * 3, workspace=True,
               scale=None, offset=(0, 0, 0)):
    size = np.dtype(NP[act]).itemsize
    bufs = [mlk.DeviceBuffer.from_array(a) for a in (q, k, v)]
    start = mlk.DeviceBuffer.from_array(batch.start)
    out = mlk.DeviceBuffer.from_array(np.full((batch.T, H, hd), 7, NP[act]))
    most = max(max(batch.counts), 1)
    need = paged.attention_packed_workspace_bytes(act, len(batch.counts), batch.T, most, H, KV, hd)
    ws = mlk.DeviceBuffer(max(need, 16), np.uint8) if workspace else None
    err = mlk.DeviceBuffer.from_array(np.zeros(1, np.int32))
    ptr = [b.offset(o * size) for b, o in zip(bufs, offset)]
    paged.attention_packed(act, *ptr, start, len(batch.counts), batch.T, most, H, KV, hd, out,
                           scale=scale, q_row_stride=strides[0], k_row_stride=strides[1],
                           v_row_stride=strides[2], workspace=ws, err=err)
    mlk.synchronize()
    assert err.download()[0] == 0
    return out.download()


def check_packed(batch, q, k, v, got, H, KV, hd, act, rows=None):
    q, k, v = (values(a, act).astype(np.float64) for a in (q, k, v))
    written = np.zeros(batch.T, bool)
    for t, s, p in batch.rows():
        written[t] = True
        if rows is not None and t not in rows:
            continue
        a = int(batch.start[s])
        kk, vv = k[a:a + p + 1], v[a:a + p + 1]
        out, pav, d = exact_rows(q[t], kk, vv, default_scale(hd))
        vsum = np.repeat(np.abs(vv).sum(0), H // KV, axis=0)
        assert_close(values(got[t], act), out, pav, d, p + 1, vsum, act, f"token {t}, sequence {s}")
    assert (got[~written] == 7).all(), "rows behind the last sequence were written"


PACKED = {
    "one": ([1], 0), "two": ([2], 0), "empty among": ([0, 3, 0, 0, 64, 1, 0], 2),
    "ragged": ([33, 1, 129, 200, 63], 1), "long": ([700], 0), "many": ([1] * 70 + [5] * 70, 0),
    "all empty": ([0, 0], 4),
}


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", list(PACKED))
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_packed_attention(mlk, paged, heads, name, act):
    H, KV, hd = heads
    counts, spare = PACKED[name]
    rng = np.random.default_rng(H * hd)
    batch = Batch(counts, None, spare=spare)
    qkv = [to_type(rng.standard_normal((batch.T, n, hd)), act) for n in (H, KV, KV)]
    for a in qkv:  # what lies behind the last sequence is not read
        a[sum(counts):] = to_type(np.float32([np.nan]), act)[0]
    got = run_packed(mlk, paged, batch, *qkv, H, KV, hd, act)
    n = sum(counts)
    some = None if H * n < 800 else set(rng.integers(0, n, 14)) | {0, n - 1}
    check_packed(batch, *qkv, got, H, KV, hd, act, rows=some)


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_packed_attention_over_a_fused_projection(mlk, paged, act, pad):
    H, KV, hd = 8, 2, 128
    batch = Batch([40, 150, 7], None, spare=1)
    rng = np.random.default_rng(4)
    width = (H + 2 * KV) * hd + pad
    qkv = to_type(rng.standard_normal((batch.T, width)), act)
    got = run_packed(mlk, paged, batch, qkv, qkv, qkv, H, KV, hd, act, strides=(width,) * 3,
                     offset=(0, H * hd, (H + KV) * hd), workspace=pad != 1)
    parts = np.split(qkv[:, :(H + 2 * KV) * hd], [H * hd, (H + KV) * hd], axis=1)
    parts = [p.reshape(batch.T, -1, hd) for p in parts]
    check_packed(batch, *parts, got, H, KV, hd, act, rows=set(range(0, 197, 9)) | {196})


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [np.inf, np.nan])
def test_packed_sequences_do_not_reach_each_other(mlk, paged, act, value):
    """One sequence of non-finite values between two others, and a non-finite
    last token."""
    H, KV, hd = 4, 2, 128
    batch = Batch([50, 20, 90], None)
    rng = np.random.default_rng(4)
    q, k, v = (rng.standard_normal((160, n, hd)).astype(np.float32) for n in (H, KV, KV))
    k[50:70], v[50:70] = value, value
    k[159], v[159] = value, value
    q, k, v = (to_type(a, act) for a in (q, k, v))
    got = run_packed(mlk, paged, batch, q, k, v, H, KV, hd, act)
    check_packed(batch, q, k, v, got, H, KV, hd, act,
                 rows=set(range(0, 50, 7)) | {49} | set(range(70, 159, 6)) | {157, 158})
    assert not np.isfinite(values(got, act)[50:70]).any()


# ------------------------------------------------------------------ append

def rope_f32(mlk, x, positions, heads, theta, neox):
    """mlk_rope_f32's result for x [T, heads, hd] (float32)."""
    T, _, hd = x.shape
    q = mlk.DeviceBuffer.from_array(np.ascontiguousarray(x))
    k = mlk.DeviceBuffer.empty((T, 1, hd))
    k.zero()
    pos = mlk.DeviceBuffer.from_array(np.asarray(positions, np.int32))
    mlk.rope(q, k, T, heads, 1, hd, positions=pos, theta=theta, rope_type=1 if neox else 0)
    return q.download()


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("heads", [(4, 2, 16), (32, 8, 128), (8, 1, 256), (5, 5, 6), (12, 12, 80),
                                   (64, 8, 128), (16, 2, 2)], ids=str)
def test_append(mlk, paged, heads, neox, act, ct):
    H, KV, hd = heads
    rng = np.random.default_rng(H + hd)
    for counts, lens, page, spare, pad, gap in (([1], [1], 16, 0, 0, 0),
                                                ([1, 0, 7, 70], [9000, 3, 7, 2000], 16, 3, 0, 0),
                                                ([20, 1], [333, 65], 1, 0, 8, 8),
                                                ([3, 2], [40, 2], 64, 1, 3, 5)):
        batch = Batch(counts, lens, page, spare)
        cache = Cache(mlk, paged, batch, KV, hd, ct, rng, gap=gap)
        width = (H + 2 * KV) * hd + pad
        qkv = to_type(rng.standard_normal((batch.T, width)), act)
        x = values(qkv, act)
        qx, kx, vx = (x[:, a * hd:b * hd].reshape(batch.T, -1, hd) for a, b in
                      ((0, H), (H, H + KV), (H + KV, H + 2 * KV)))
        pos = np.zeros(batch.T, np.int32)
        for t, s, p in batch.rows():
            pos[t] = p
        dev = batch.device(mlk, paged)
        buf = mlk.DeviceBuffer.from_array(qkv)
        size = qkv.itemsize
        q_out = mlk.DeviceBuffer.from_array(np.full((batch.T, H, hd), 7, NP[act]))
        err = mlk.DeviceBuffer.from_array(np.zeros(1, np.int32))
        paged.kv_append(cache.handle, dev, buf.offset(H * hd * size),
                        buf.offset((H + KV) * hd * size), act, q=buf, q_out=q_out, n_heads=H,
                        theta=5e5, rope_type=int(neox), q_row_stride=width, k_row_stride=width,
                        v_row_stride=width, err=err)
        mlk.synchronize()
        assert err.download()[0] == 0
        assert (buf.download() == qkv).all()
        want_q = to_type(rope_f32(mlk, qx, pos, H, 5e5, neox), act)
        want_k = to_type(rope_f32(mlk, kx, pos, KV, 5e5, neox), ct)
        want_q[int(batch.start[-1]):] = 7
        hosts = [a.copy() for a in cache.host]
        for t, s, p in batch.rows():
            pg, r = batch.table[s, p // page], p % page
            cache.pages(0, hosts[0])[pg, r] = want_k[t]
            cache.pages(1, hosts[1])[pg, r] = to_type(vx[t], ct)
        same = lambda a, b: np.array_equal(a.view(np.uint8), b.view(np.uint8))  # noqa: E731
        assert same(q_out.download(), want_q)
        assert same(cache.k.download(), hosts[0]) and same(cache.v.download(), hosts[1])
        # in place, without q, and unrotated
        paged.kv_append(cache.handle, dev, buf.offset(H * hd * size),
                        buf.offset((H + KV) * hd * size), act, q=buf, n_heads=H, theta=5e5,
                        rope_type=int(neox), q_row_stride=width, k_row_stride=width,
                        v_row_stride=width)
        after = buf.download()
        n = int(batch.start[-1])
        assert same(np.ascontiguousarray(after[:n, :H * hd]),
                    np.ascontiguousarray(want_q.reshape(batch.T, -1)[:n]))
        assert same(np.ascontiguousarray(after[:, H * hd:]),
                    np.ascontiguousarray(qkv[:, H * hd:]))
        assert same(np.ascontiguousarray(after[n:]), np.ascontiguousarray(qkv[n:]))
        paged.kv_append(cache.handle, dev, buf.offset(H * hd * size),
                        buf.offset((H + KV) * hd * size), act, theta=0.0, k_row_stride=width,
                        v_row_stride=width)
        for t, s, p in batch.rows():
            cache.pages(0, hosts[0])[batch.table[s, p // page], p % page] = to_type(kx[t], ct)
        assert same(cache.k.download(), hosts[0]) and same(cache.v.download(), hosts[1])


def test_append_odd_head_dim_without_rotation(mlk, paged):
    H, KV, hd = 1, 3, 5
    batch = Batch([4, 2], [9, 2], 4)
    rng = np.random.default_rng(0)
    for act, ct in PAIRS:
        cache = Cache(mlk, paged, batch, KV, hd, ct, rng)
        k, v = (to_type(rng.standard_normal((batch.T, KV, hd)), act) for _ in range(2))
        paged.kv_append(cache.handle, batch.device(mlk, paged), mlk.DeviceBuffer.from_array(k),
                        mlk.DeviceBuffer.from_array(v), act, theta=0.0)
        mlk.synchronize()
        for t, s, p in batch.rows():
            cache.pages(0)[batch.table[s, p // 4], p % 4] = to_type(values(k[t], act), ct)
            cache.pages(1)[batch.table[s, p // 4], p % 4] = to_type(values(v[t], act), ct)
        assert (cache.k.download().view(np.uint8) == cache.host[0].view(np.uint8)).all()
        assert (cache.v.download().view(np.uint8) == cache.host[1].view(np.uint8)).all()


# ------------------------------------------------------------------ wrong values on the device

def test_bad_pages_and_sequences_raise_the_flag(mlk, paged):
    """Page indexes outside the cache and sequences outside the bounds: the
    flag, nothing written for them, the other sequences as ever."""
    H, KV, hd = 8, 2, 64
    rng = np.random.default_rng(2)
    for act, ct in PAIRS:
        for what in ("page", "negative page", "too many", "too long", "more than its length",
                     "beyond the rows"):
            batch = Batch([3, 2, 30], [40, 20, 35], 16)
            cache = Cache(mlk, paged, batch, KV, hd, ct, rng)
            good_table, good_start = batch.table.copy(), batch.start.copy()
            max_new, max_len = 30, 40
            lens = list(batch.lens)
            if what == "page":
                batch.table[1, 1] = batch.n_pages
            elif what == "negative page":
                batch.table[1, 1] = -5
            elif what == "too many":
                max_new, wrong = 29, 2
            elif what == "too long":
                batch.lens[1] = 41
            elif what == "more than its length":
                batch.lens[1] = 1
            else:
                batch.start[-1] = batch.T + 1
            wrong = 1 if "page" in what or batch.lens[1] != 20 else 2
            dev = batch.device(mlk, paged, max_new, max_len)
            batch.table, batch.start, batch.lens = good_table, good_start, lens
            q = to_type(rng.standard_normal((batch.T, H, hd)), act)
            dq = mlk.DeviceBuffer.from_array(q)
            out = mlk.DeviceBuffer.from_array(np.full((batch.T, H, hd), 7, NP[act]))
            err = mlk.DeviceBuffer.from_array(np.zeros(1, np.int32))
            paged.attention(cache.handle, dev, dq, out, H, act, err=err)
            mlk.synchronize()
            assert err.download()[0] != 0, what
            got = out.download()
            rows = [t for t, s, p in batch.rows() if s != wrong]
            part = [t for t, s, p in batch.rows() if s == wrong]
            if "page" not in what:
                assert (got[part] == 7).all(), what
            check_paged(batch, cache, q, got, H, act, rows=set(rows))
            # append: the rows of that page, or the sequence, stay as they were
            k = to_type(rng.standard_normal((batch.T, KV, hd)), act)
            err.zero()
            before = [a.copy() for a in cache.host]
            paged.kv_append(cache.handle, dev, mlk.DeviceBuffer.from_array(k),
                            mlk.DeviceBuffer.from_array(k), act, theta=0.0, err=err)
            mlk.synchronize()
            assert err.download()[0] != 0, what
            for t, s, p in batch.rows():
                if s != wrong:
                    for a in before:
                        cache.pages(0, a)[batch.table[s, p // 16], p % 16] = \
                            to_type(values(k[t], act), ct)
            for b, a in zip((cache.k, cache.v), before):
                assert (b.download().view(np.uint8) == a.view(np.uint8)).all(), what


# ------------------------------------------------------------------ as they are used

@pytest.mark.parametrize("act,ct", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
def test_prompts_then_decode_steps(mlk, paged, act, ct):
    """Two prompts through packed attention and the append, a chunk, then
    decode steps: every output against float64 over the whole history, and
    for fp32 against the contiguous cache's own entries."""
    H, KV, hd, page, theta = 8, 2, 64, 16, 1e4
    rng = np.random.default_rng(8)
    final = [90, 61]
    plan = Batch([1, 1], final, page)
    cache = Cache(mlk, paged, plan, KV, hd, ct, rng, fill=False)
    done = [0, 0]
    hist = [[], []]  # rotated k and v rows as the cache holds them
    for counts in ([50, 23], [17, 36], [1, 1], [1, 0], [21, 1]):
        lens = [d + c for d, c in zip(done, counts)]
        batch = Batch(counts, [max(n, 1) for n in lens], page)
        batch.table, batch.n_pages, batch.width = plan.table, plan.n_pages, plan.width
        T = batch.T
        x = [to_type(rng.standard_normal((T, n, hd)), act) for n in (H, KV, KV)]
        pos = np.zeros(T, np.int32)
        for t, s, p in batch.rows():
            pos[t] = p
        d = [mlk.DeviceBuffer.from_array(a) for a in x]
        dev = batch.device(mlk, paged)
        paged.kv_append(cache.handle, dev, d[1], d[2], act, q=d[0], n_heads=H, theta=theta)
        out = mlk.DeviceBuffer.empty((T, H, hd), NP[act])
        ws = mlk.DeviceBuffer(max(16, paged.attention_workspace_bytes(cache.handle, dev, H)),
                              np.uint8)
        paged.attention(cache.handle, dev, d[0], out, H, act, workspace=ws)
        mlk.synchronize()
        got = out.download()
        qr = to_type(rope_f32(mlk, values(x[0], act), pos, H, theta, False), act)
        kr = to_type(rope_f32(mlk, values(x[1], act), pos, KV, theta, False), ct)
        for t, s, p in batch.rows():
            hist[s].append((values(kr[t], ct), values(to_type(values(x[2][t], act), ct), ct)))
        for t, s, p in batch.rows():
            k, v = (np.array([h[i] for h in hist[s][:p + 1]], np.float64) for i in range(2))
            o, pav, dd = exact_rows(values(qr[t], act).astype(np.float64), k, v, default_scale(hd))
            vsum = np.repeat(np.abs(v).sum(0), H // KV, axis=0)
            assert_close(values(got[t], act), o, pav, dd, p + 1, vsum, act, f"token {t}")
        if not any(done) and act == ct:  # whole prompts: the packed form on the same rows
            kp, vp = (mlk.DeviceBuffer.from_array(a) for a in (kr, to_type(values(x[2], act), ct)))
            st = mlk.DeviceBuffer.from_array(batch.start)
            o2 = mlk.DeviceBuffer.empty((T, H, hd), NP[act])
            paged.attention_packed(act, d[0], kp, vp, st, 2, T, 50, H, KV, hd, o2)
            mlk.synchronize()
            check_packed(Batch(counts, None), qr, kr, to_type(values(x[2], act), ct),
                         o2.download(), H, KV, hd, act)
        if act == ct == "f32":
            for s in range(2):
                rows = [t for t, r, p in batch.rows() if r == s]
                if not rows:
                    continue
                kc, vc = (mlk.DeviceBuffer.from_array(np.array([h[i] for h in hist[s]],
                                                               np.float32)) for i in range(2))
                o3 = mlk.DeviceBuffer.empty((len(rows), H, hd))
                dq = mlk.DeviceBuffer.from_array(qr[rows])
                n = lens[s]
                w = mlk.DeviceBuffer(max(16, mlk.attention_workspace_bytes(len(rows), H, KV, hd,
                                                                           n)), np.uint8)
                mlk.attention_decode(dq, kc, vc, 1, n, H, KV, hd, 0, len(rows), o3, n,
                                     pos0=n - len(rows), workspace=w, workspace_bytes=w.nbytes)
                assert np.abs(o3.download() - got[rows]).max() <= 4e-5
        done = lens


def test_captured_step_replays_with_new_lengths(mlk, paged):
    """Append and attention captured once; the metadata, inputs and padded
    tokens change between replays; two graphs share a workspace on one
    stream."""
    H, KV, hd, page = 8, 2, 64, 16
    rng = np.random.default_rng(6)
    plan = Batch([40, 4, 4], [700, 300, 260], page)
    cache = Cache(mlk, paged, plan, KV, hd, "f16", rng)
    dev = plan.device(mlk, paged, max_new=40, max_len=700)
    T = plan.T
    bufs = [mlk.DeviceBuffer.empty((T, n, hd)) for n in (H, KV, KV)]
    out = mlk.DeviceBuffer.empty((T, H, hd))
    ws = mlk.DeviceBuffer(max(16, paged.attention_workspace_bytes(cache.handle, dev, H)), np.uint8)
    stream = mlk.Stream()
    graphs = []
    for _ in range(2):
        with mlk.Graph.capture(stream) as g:
            paged.kv_append(cache.handle, dev, bufs[1], bufs[2], "f32", theta=0.0, stream=stream)
            paged.attention(cache.handle, dev, bufs[0], out, H, "f32", workspace=ws, stream=stream)
        graphs.append(g)
    for step, (counts, lens) in enumerate((([40, 4, 4], [700, 300, 260]), ([1, 1, 1], [600, 1, 40]),
                                           ([33, 0, 9], [33, 299, 255]), ([2, 3, 1], [5, 290, 20]))):
        now = Batch(counts, lens, page, spare=T - sum(counts))
        now.table, now.n_pages = plan.table, plan.n_pages
        plan.keep[0].upload(now.start)
        plan.keep[1].upload(np.asarray(lens, np.int32))
        x = [rng.standard_normal((T, n, hd)).astype(np.float32) for n in (H, KV, KV)]
        for b, a in zip(bufs, x):
            b.upload(a)
        out.upload(np.full((T, H, hd), 7, np.float32))
        mlk.synchronize()
        graphs[step % 2].launch()
        stream.synchronize()
        for t, s, p in now.rows():
            pg, r = now.table[s, p // page], p % page
            cache.pages(0)[pg, r], cache.pages(1)[pg, r] = x[1][t], x[2][t]
        cache.batch = now
        check_paged(now, cache, x[0], out.download(), H, "f32")
        mlk.synchronize()


def test_two_streams_at_once(mlk, paged):
    """Calls on two streams with a workspace each: each as alone, bit for bit."""
    H, KV, hd = 32, 8, 128
    rng = np.random.default_rng(7)
    batch = Batch([1, 1], [5000, 3000], 16)
    cache = Cache(mlk, paged, batch, KV, hd, "f16", rng)
    q = [rng.standard_normal((2, H, hd)).astype(np.float32) for _ in range(2)]
    want = [run_paged(mlk, paged, batch, cache, a, H, "f32") for a in q]
    dev = batch.device(mlk, paged)
    streams = [mlk.Stream() for _ in range(2)]
    dq = [mlk.DeviceBuffer.from_array(a) for a in q]
    outs = [mlk.DeviceBuffer.empty((2, H, hd)) for _ in q]
    need = max(16, paged.attention_workspace_bytes(cache.handle, dev, H))
    wss = [mlk.DeviceBuffer(need, np.uint8) for _ in q]
    for _ in range(5):
        for i in range(2):
            paged.attention(cache.handle, dev, dq[i], outs[i], H, "f32", workspace=wss[i],
                            stream=streams[i])
    for s in streams:
        s.synchronize()
    for o, w in zip(outs, want):
        assert (o.download() == w).all()


def test_cache_beyond_32_bit_offsets(mlk, paged):
    """Pages over 4 GiB (and 2^31 elements) into the buffers, fp32 and 16-bit."""
    H, KV, hd, page = 4, 1, 128, 64
    row = page * KV * hd
    for act, ct, stride in (("f32", "f16", 1 << 26), ("f32", "f32", 1 << 25),
                            ("bf16", "bf16", 1 << 26)):
        n_pages = 70
        size = np.dtype(NP[ct]).itemsize
        bufs = [mlk.DeviceBuffer(((n_pages - 1) * stride + row) * size, NP[ct]) for _ in range(2)]
        handle = paged.PagedCache(*bufs, ct, n_pages, page, KV, hd, page_stride=stride)
        batch = Batch([5], [200], page)
        batch.table[0, :4] = [69, 0, 68, 33]
        batch.n_pages = n_pages
        rng = np.random.default_rng(1)
        k, v = (to_type(rng.standard_normal((200, KV, hd)), ct) for _ in range(2))
        for j in range(4):
            n = min(page, 200 - j * page)
            for b, a in zip(bufs, (k, v)):
                part = np.ascontiguousarray(a[j * page:j * page + n])
                mlk.check(mlk.lib.mlk_memcpy(b.offset(int(batch.table[0, j]) * stride * size),
                                             part.ctypes.data, part.nbytes, mlk.H2D))
        q = to_type(rng.standard_normal((5, H, hd)), act)
        dev = batch.device(mlk, paged)
        out = mlk.DeviceBuffer.empty((5, H, hd), NP[act])
        kn, vn = (np.ascontiguousarray(a[195:]) for a in (k, v))
        if act == ct:  # append the last five rows again, unrotated
            paged.kv_append(handle, dev, mlk.DeviceBuffer.from_array(kn),
                            mlk.DeviceBuffer.from_array(vn), act, theta=0.0)
        paged.attention(handle, dev, mlk.DeviceBuffer.from_array(q), out, H, act)
        mlk.synchronize()
        k64, v64 = (values(a, ct).astype(np.float64) for a in (k, v))
        got = values(out.download(), act)
        for i in range(5):
            n = 196 + i
            o, pav, d = exact_rows(values(q[i], act).astype(np.float64), k64[:n], v64[:n],
                                   default_scale(hd))
            vsum = np.repeat(np.abs(v64[:n]).sum(0), H, axis=0)
            assert_close(got[i], o, pav, d, n, vsum, act, f"row {i}")


# ------------------------------------------------------------------ many sequences, odd tables

@pytest.mark.parametrize("act,ct", PAIRS)
def test_more_sequences_than_a_wave(mlk, paged, act, ct):
    """150 sequences: decode steps, a mixed batch with empty ones, and packed
    prompts; some of them longer than what is left unsplit."""
    H, KV, hd = 8, 2, 64
    rng = np.random.default_rng(11)
    lens = rng.integers(1, 90, 150)
    lens[[3, 64, 149]] = 1200, 700, 2001
    for counts in (np.ones(150, int), np.where(np.arange(150) % 7 == 2, 0, 1)):
        counts = counts.copy()
        if counts.sum() < 150:
            counts[[3, 77, 149]] = 9, 21, 300
        lens = np.maximum(lens, counts)
        batch = Batch(counts, lens, 16, spare=1, seed=3)
        cache = Cache(mlk, paged, batch, KV, hd, ct, rng)
        q = to_type(rng.standard_normal((batch.T, H, hd)), act)
        got = run_paged(mlk, paged, batch, cache, q, H, act)
        some = set(rng.integers(0, sum(counts), 60)) | {0, 3, 4, 20, 64, sum(counts) - 1}
        check_paged(batch, cache, q, got, H, act, rows=some)
    if act == ct:
        batch = Batch(np.minimum(lens, 90), None)
        qkv = [to_type(rng.standard_normal((batch.T, n, hd)), act) for n in (H, KV, KV)]
        got = run_packed(mlk, paged, batch, *qkv, H, KV, hd, act)
        check_packed(batch, *qkv, got, H, KV, hd, act, rows=set(rng.integers(0, batch.T, 60)))


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("page", [2, 4, 8, 32])
@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 8, 128), (4, 1, 160), (4, 2, 72)], ids=str)
def test_page_sizes(mlk, paged, heads, page, act, ct):
    H, KV, hd = heads
    rng = np.random.default_rng(page)
    for counts, lens in (([1, 1, 1], [777, 64, 33]), ([40, 1], [700, 130])):
        batch = Batch(counts, lens, page, seed=page)
        cache = Cache(mlk, paged, batch, KV, hd, ct, rng)
        q = to_type(rng.standard_normal((batch.T, H, hd)), act)
        got = run_paged(mlk, paged, batch, cache, q, H, act)
        check_paged(batch, cache, q, got, H, act, rows=set(range(0, batch.T, 5)) | {batch.T - 1})


@pytest.mark.parametrize("act,ct", [("f32", "f16"), ("bf16", "bf16")])
def test_shared_pages_dirty_workspace_and_no_flag(mlk, paged, act, ct):
    """Two sequences on the same first pages; a workspace full of NaN bits, used
    by two calls of different sizes; err not given."""
    H, KV, hd, page = 8, 2, 128, 16
    rng = np.random.default_rng(12)
    batch = Batch([1, 1], [1000, 900], page)
    shared = 800 // page
    batch.table[1, :shared] = batch.table[0, :shared]
    cache = Cache(mlk, paged, batch, KV, hd, ct, rng)
    dev = batch.device(mlk, paged)
    need = paged.attention_workspace_bytes(cache.handle, dev, H, act)
    assert need > 0
    ws = mlk.DeviceBuffer.from_array(np.full(need, 0xFF, np.uint8))
    q = to_type(rng.standard_normal((2, H, hd)), act)
    for b in (batch, Batch([1], [600], page)):
        b.table, b.n_pages, b.width = batch.table, batch.n_pages, batch.width
        d = b.device(mlk, paged)
        out = mlk.DeviceBuffer.from_array(np.full((b.T, H, hd), 7, NP[act]))
        paged.attention(cache.handle, d, mlk.DeviceBuffer.from_array(q[:b.T].copy()), out, H, act,
                        workspace=ws)
        mlk.synchronize()
        cache.batch = b
        check_paged(b, cache, q[:b.T], out.download(), H, act)


def test_split_results_do_not_depend_on_the_bounds(mlk, paged):
    """Host bounds far above the lengths: the same values to rounding, with the
    workspace such bounds ask for."""
    H, KV, hd = 32, 8, 128
    rng = np.random.default_rng(13)
    for counts, lens in (([1, 1], [900, 40]), ([70], [800])):
        batch = Batch(counts, lens, 16)
        cache = Cache(mlk, paged, batch, KV, hd, "f16", rng)
        batch.table = np.pad(batch.table, ((0, 0), (0, 2000)), constant_values=-1)
        batch.width = batch.table.shape[1]
        q = rng.standard_normal((batch.T, H, hd)).astype(np.float32)
        for bounds in ((None, None), (batch.T, 30000)):
            dev = batch.device(mlk, paged, *bounds)
            got = run_paged(mlk, paged, batch, cache, q, H, "f32", dev=dev)
            check_paged(batch, cache, q, got, H, "f32", rows=set(range(0, batch.T, 9)))


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 8, 128), (4, 1, 160)], ids=str)
def test_more_sequences_than_workgroups(mlk, paged, heads, act, ct):
    """700 sequences, few of them long enough to be split, some without a new
    token: those that lie across two workgroups' shares are joined, and only
    those; the same again without a workspace."""
    H, KV, hd = heads
    rng = np.random.default_rng(21)
    lens = [int(n) for n in rng.integers(1, 41, 700)]
    for s in range(13, 700, 60):
        lens[s] = int(rng.integers(600, 1500))
    counts = [0 if s % 9 == 4 else 1 for s in range(700)]
    batch = Batch(counts, lens, 16, 2)
    cache = Cache(mlk, paged, batch, KV, hd, ct, rng)
    q = to_type(rng.standard_normal((batch.T, H, hd)), act)
    rows = {t for t, s, p in batch.rows() if lens[s] > 500 or s % 17 == 0}
    for ws in (True, False):
        got = run_paged(mlk, paged, batch, cache, q, H, act, workspace=ws)
        check_paged(batch, cache, q, got, H, act, rows=rows)
        g = values(got[:sum(counts)], act)
        assert np.isfinite(g).all() and (g != 7).any(axis=(1, 2)).all()


def test_thousands_of_sequences(mlk, paged):
    """5000 sequences of 0, 1 or 2 new tokens, one of 40: each token's place in
    its own sequence's pages, and packed attention within its own sequence."""
    H, KV, hd = 4, 1, 16
    rng = np.random.default_rng(22)
    counts = [int(n) for n in rng.integers(0, 3, 5000)]
    counts[4321] = 40
    batch = Batch(counts, [n + s % 3 + 1 for s, n in enumerate(counts)], 2, 3)
    cache = Cache(mlk, paged, batch, KV, hd, "f32", rng, fill=False)
    q, k, v = (rng.standard_normal((batch.T, n, hd)).astype(np.float32) for n in (H, KV, KV))
    err = mlk.DeviceBuffer.from_array(np.zeros(1, np.int32))
    paged.kv_append(cache.handle, batch.device(mlk, paged), mlk.DeviceBuffer.from_array(k),
                    mlk.DeviceBuffer.from_array(v), "f32", theta=0.0, err=err)
    mlk.synchronize()
    assert err.download()[0] == 0
    for t, s, p in batch.rows():
        cache.pages(0)[batch.table[s, p // 2], p % 2] = k[t]
        cache.pages(1)[batch.table[s, p // 2], p % 2] = v[t]
    assert (cache.k.download().view(np.uint8) == cache.host[0].view(np.uint8)).all()
    assert (cache.v.download().view(np.uint8) == cache.host[1].view(np.uint8)).all()
    packed = Batch(counts, None, spare=3)
    got = run_packed(mlk, paged, packed, q, k, v, H, KV, hd, "f32")
    at = int(packed.start[4321])
    check_packed(packed, q, k, v, got, H, KV, hd, "f32",
                 rows=set(range(0, sum(counts), 23)) | set(range(at, at + 42)))


def test_mixed_batch_of_very_many_sequences(mlk, paged):
    """70000 decode tokens on two shared pages and a chunk of 40 beside them,
    under a bound of 8192 positions: too many row tiles for as many parts as the
    chunk alone would be split into."""
    H, KV, hd = 8, 8, 8
    rng = np.random.default_rng(23)
    lens = [int(n) for n in rng.integers(1, 6, 70000)] + [700]
    batch = Batch([1] * 70000 + [40], lens, 8192)
    batch.n_pages = 2
    batch.table[:, 0] = np.arange(len(lens)) % 2
    cache = Cache(mlk, paged, batch, KV, hd, "bf16", rng)
    q = to_type(rng.standard_normal((batch.T, H, hd)), "bf16")
    got = run_paged(mlk, paged, batch, cache, q, H, "bf16",
                    dev=batch.device(mlk, paged, None, 8192))
    check_paged(batch, cache, q, got, H, "bf16",
                rows=set(range(0, 70000, 997)) | set(range(69995, 70040, 3)))


# ------------------------------------------------------------------ large scores

PLANS = {  # new tokens, lengths, workspace: which kernel, positions split or not
    "few": ([1, 3], [300, 90], False),
    "few split": ([1, 1, 1], [3000, 700, 20], True),
    "tile": ([40], [190], False),
    "tile split": ([40], [3000], True),
    "both": ([40, 1, 1], [1200, 900, 30], True),
}


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("name", list(PLANS))
@pytest.mark.parametrize("hd,scale", [(128, None), (128, 1.0), (64, None)])
def test_large_finite_scores(mlk, paged, hd, scale, name, act, ct):
    """Every key alike but one per KV head, which all of q prefers by far: a token
    before it gets the mean of V so far, the others its V row.  Equal keys give
    bit-equal scores and the others differ by far more than a score's rounding, so
    the error of a score, however large the scores are, is no part of the bound."""
    H, KV = 8, 2
    counts, lens, ws = PLANS[name]
    rng = np.random.default_rng(31)
    batch = Batch(counts, lens, 16, seed=2)
    for x in (1448, 1700, 2222, 4000) if "f16" in (act, ct) else (17000, 20000, 50000, 1000000):
        cache = Cache(mlk, paged, batch, KV, hd, ct, rng)
        for s, n in enumerate(lens):
            pg, r = batch.slots(s, n)
            cache.pages(0)[pg, r] = to_type(np.float32([-x]), ct)[0]
            for g, j in ((0, n - 1 - counts[s] // 2), (1, n // 3)):
                cache.pages(0)[pg[j], r[j], g] = to_type(np.float32([x]), ct)[0]
        cache.upload(mlk)
        cache.handle = paged.PagedCache(cache.k, cache.v, ct, batch.n_pages, batch.page, KV, hd)
        q = to_type(np.full((batch.T, H, hd), x, np.float32), act)
        got = run_paged(mlk, paged, batch, cache, q, H, act, scale=scale, workspace=ws)
        q64 = values(q, act).astype(np.float64)
        for t, s, p in batch.rows():
            if t % 3 and p + 1 < lens[s]:
                continue
            k, v = (a[:p + 1] for a in cache.gathered(s, lens[s]))
            out, pav, _ = exact_rows(q64[t], k, v, scale or default_scale(hd))
            vsum = np.repeat(np.abs(v).sum(0), H // KV, axis=0)
            assert_close(values(got[t], act), out, pav, 0.0, p + 1, vsum, act,
                         f"{x}: token {t} (sequence {s}, position {p})")


# ------------------------------------------------------------------ wrong values where positions are split

SPLITS = {  # H, KV, hd, page, new tokens, lengths, sequences that a wrong value is put into
    "few, page 2": (8, 2, 64, 2, [1, 1, 1, 1], [3000, 700, 20, 900], [0, 1, 2]),
    "few, page 8": (8, 2, 64, 8, [3, 1, 2, 1], [3000, 700, 20, 900], [0, 2]),
    "few, page 16": (8, 2, 128, 16, [1, 1, 2], [2000, 1500, 1300], [1]),
    "few, a wave a head": (16, 8, 64, 16, [1] * 40, [1700] * 40, [0, 17, 39]),
    "few, by worker": (8, 8, 64, 16, [0 if s % 9 == 4 else 1 for s in range(700)],
                       [1200 if s % 60 == 13 else 1 + s % 40 for s in range(700)], [13, 73, 300]),
    "tile": (8, 2, 64, 16, [40, 60], [3000, 1500], [0, 1]),
    "tile, page 2": (8, 2, 128, 2, [70, 0, 9], [2000, 30, 600], [0]),
    "both": (8, 2, 64, 16, [40, 1, 1, 0, 1], [2500, 1500, 30, 20, 1100], [0, 1]),
}


@pytest.mark.parametrize("act,ct", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("name", list(SPLITS))
def test_bad_pages_and_sequences_where_positions_are_split(mlk, paged, name, act, ct):
    """Page indexes outside the cache and sequences outside the bounds, through
    every form of the page look-up, the division of work and the joins: the flag,
    nothing written for a refused sequence, the others as ever."""
    H, KV, hd, page, counts, lens, where = SPLITS[name]
    rng = np.random.default_rng(41)
    batch = Batch(counts, lens, page, spare=2, seed=5)
    cache = Cache(mlk, paged, batch, KV, hd, ct, rng)
    q = to_type(rng.standard_normal((batch.T, H, hd)), act)
    good_table, good_lens = batch.table.copy(), list(batch.lens)
    rows = list(batch.rows())
    for wrong in where:
        n = lens[wrong]
        for what in ("first page", "middle page", "last page", "too long", "more than its length"):
            batch.table, batch.lens = good_table.copy(), list(good_lens)
            if what == "too long":
                batch.lens[wrong] = max(lens) + 1
            elif what == "more than its length":
                batch.lens[wrong] = counts[wrong] - 1
            else:
                at = {"first page": 0, "middle page": (n - 1) // page // 2,
                      "last page": (n - 1) // page}[what]
                batch.table[wrong, at] = -7 if wrong % 2 else batch.n_pages
            dev = batch.device(mlk, paged, max(counts), max(lens))
            batch.table, batch.lens = good_table, good_lens
            need = paged.attention_workspace_bytes(cache.handle, dev, H, act)
            assert need > 0
            ws = mlk.DeviceBuffer.from_array(np.full(need, 0xFF, np.uint8))
            out = mlk.DeviceBuffer.from_array(np.full((batch.T, H, hd), 7, NP[act]))
            err = mlk.DeviceBuffer.from_array(np.zeros(1, np.int32))
            paged.attention(cache.handle, dev, mlk.DeviceBuffer.from_array(q), out, H, act,
                            workspace=ws, err=err)
            mlk.synchronize()
            # (pages of a sequence without a new token are not looked at)
            assert (err.download()[0] != 0) == (counts[wrong] > 0 or "page" not in what), what
            got = out.download()
            if "page" not in what:
                assert (got[[t for t, s, p in rows if s == wrong]] == 7).all(), what
            others = [t for t, s, p in rows if s != wrong]
            assert (got[others] != 7).any(axis=(1, 2)).all(), what
            check_paged(batch, cache, q, got, H, act, rows=set(others[::1 + len(others) // 9]))


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("name", ["few, page 8", "few, a wave a head", "tile", "tile, page 2", "both"])
def test_non_finite_values_where_positions_are_split(mlk, paged, name, act, ct):
    """A non-finite V or K, met in a fully or partly masked tile of one part of a
    row: the rows that attend to it non-finite in its dims, all others as without."""
    H, KV, hd, page, counts, lens, _ = SPLITS[name]
    rng = np.random.default_rng(43)
    counts = [3] * len(counts) if name == "few, a wave a head" else counts
    batch = Batch(counts, lens, page, seed=6)
    cache = Cache(mlk, paged, batch, KV, hd, ct, rng)
    q = to_type(rng.standard_normal((batch.T, H, hd)), act)
    good = [a.copy() for a in cache.host]
    n, c = lens[0], counts[0]
    pg, r = batch.slots(0, n)
    for pos in (n - 2, n - c // 2 - 1, n - c - 1, n // 2, 257, 0):
        for which, value in ((1, np.inf), (1, -np.inf), (1, np.nan), (0, np.nan)):
            dims = slice(hd // 2, hd // 2 + 3) if which else slice(0, hd)
            cache.host = [a.copy() for a in good]
            cache.pages(which)[pg[pos], r[pos], 1, dims] = to_type(np.float32([value]), ct)[0]
            cache.upload(mlk)
            cache.handle = paged.PagedCache(cache.k, cache.v, ct, batch.n_pages, batch.page, KV, hd)
            got = run_paged(mlk, paged, batch, cache, q, H, act)
            what = f"position {pos}, {'KV'[which]} {value}"
            g = values(got, act).reshape(batch.T, KV, H // KV, hd)
            first = n - c  # token row t of sequence 0 is at position first + t
            sees = [t for t in range(c) if first + t >= pos]
            assert not np.isfinite(g[sees, 1][..., dims]).any(), what
            g = g.copy()
            g[sees, 1, :, dims] = 0
            assert np.isfinite(g).all(), what
            others = [t for t, s, p in batch.rows() if s != 0 or p < pos]
            check_paged(batch, cache, q, got, H, act, rows=set(others[-7:] + others[:2]))


# ------------------------------------------------------------------ more workgroups than a launch takes

@pytest.mark.parametrize("chunk,max_len,workspace", [(1, 512, True), (1, 513, True), (1, 513, False),
                                                     (40, 512, True), (40, 513, False)])
def test_more_workgroups_than_a_launch(mlk, paged, chunk, max_len, workspace):
    """600000 sequences at 8 KV heads, 4.8 million (sequence, head) pairs, on two
    shared pages: run whether the lengths' bound lets them be split or not, with and
    without a workspace, with one token each and beside a chunk."""
    H, KV, hd, n = 8, 8, 8, 600000
    rng = np.random.default_rng(51)
    lens = rng.integers(1, 6, n)
    counts = np.ones(n, int)
    lens[n // 2], counts[n // 2] = 500, chunk
    batch = Batch([1], [1024], 1024)
    batch.counts, batch.lens = counts.tolist(), lens.tolist()
    batch.start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    batch.T, batch.n_pages = int(batch.start[-1]), 2
    batch.table = (np.arange(n) % 2).astype(np.int32).reshape(n, 1)
    cache = Cache(mlk, paged, batch, KV, hd, "bf16", rng, fill=False)
    for i in range(2):
        cache.host[i] = to_type(rng.standard_normal(cache.host[i].shape), "bf16")
    cache.upload(mlk)
    cache.handle = paged.PagedCache(cache.k, cache.v, "bf16", 2, 1024, KV, hd)
    q = to_type(rng.standard_normal((batch.T, H, hd)), "bf16")
    got = run_paged(mlk, paged, batch, cache, q, H, "bf16", workspace=workspace,
                    dev=batch.device(mlk, paged, chunk, max_len))
    assert (got != 7).any(axis=(1, 2)).all()
    at = int(batch.start[n // 2])
    check_paged(batch, cache, q, got, H, "bf16",
                rows=set(range(0, n, 4999)) | set(range(524280, 524296)) | {at, batch.T - 1})


# ------------------------------------------------------------------ few rows: weights of 16-bit activations

FEW = {  # new tokens, lengths, workspace; 8 KV heads over many sequences: a wave to a head
    "one": ([1, 2, 1], [24, 300, 33], 2, False),
    "split": ([1, 1, 2], [40, 2000, 700], 2, True),
    "a wave a head": ([1] * 40, [700] * 40, 8, True),
}


@pytest.mark.parametrize("act", ["f16", "bf16"])
@pytest.mark.parametrize("name", list(FEW))
@pytest.mark.parametrize("hd", [64, 128])
def test_few_rows_keep_the_weights_of_16_bit_activations(mlk, paged, hd, name, act):
    """Scores that are exact (whole numbers times a power of two), so that what is
    left is the weights' precision: two pieces, 2^-15 of a weight (bf16), 2^-20 and
    2^-37 of the largest (fp16), not one rounding to the type (2^-9, 2^-12).  The
    rest as in paged_cases.py: exp, sum and division (n + 54) u, the result's own
    rounding."""
    counts, lens, KV, ws = FEW[name]
    H = 2 * KV
    rng = np.random.default_rng(61)
    batch = Batch(counts, lens, 16, seed=8)
    cache = Cache(mlk, paged, batch, KV, hd, act, rng)
    for s, n in enumerate(lens):
        pg, r = batch.slots(s, n)
        cache.pages(0)[pg, r] = to_type(rng.integers(-1, 2, (n, KV, hd)), act)
    cache.upload(mlk)
    cache.handle = paged.PagedCache(cache.k, cache.v, act, batch.n_pages, batch.page, KV, hd)
    q = to_type(rng.choice([-1.0, 1.0], (batch.T, H, hd)), act)
    got = values(run_paged(mlk, paged, batch, cache, q, H, act, scale=1 / 16, workspace=ws), act)
    e, least = (2.0 ** -15, 0.0) if act == "bf16" else (2.0 ** -20, 2.0 ** -37)
    half, tiny = 2.0 ** -8 if act == "bf16" else 2.0 ** -11, 2.0 ** -25 if act == "f16" else 0.0
    for t, s, p in batch.rows():
        if t % 5 and s < len(lens) - 1:
            continue
        k, v = (a[:p + 1] for a in cache.gathered(s, lens[s]))
        out, pav, _ = exact_rows(values(q[t], act).astype(np.float64), k, v, 1 / 16)
        vsum = np.repeat(np.abs(v).sum(0), H // KV, axis=0)
        bound = ((p + 55) * 2.0 ** -24 + e) * pav + least * vsum
        bound = bound + half * (np.abs(out) + bound) + tiny
        err = np.abs(got[t].astype(np.float64) - out)
        assert (err <= bound).all(), (f"token {t}: {int((err > bound).sum())} of {err.size}, "
                                      f"{float((err / bound).max()):.2f} of the bound")


@pytest.mark.parametrize("act", ["f16", "bf16"])
@pytest.mark.parametrize("name", list(FEW))
@pytest.mark.parametrize("value", [np.inf, -np.inf])
@pytest.mark.parametrize("equal", [False, True])
def test_few_rows_keep_an_infinity(mlk, paged, equal, value, name, act):
    """An infinity in V in a tile that every row attends to, of 16-bit activations:
    itself, also where the weights are powers of two."""
    counts, lens, KV, ws = FEW[name]
    H, hd = 2 * KV, 64
    rng = np.random.default_rng(62)
    batch = Batch(counts, lens, 16, seed=9)
    cache = Cache(mlk, paged, batch, KV, hd, act, rng)
    pg, r = batch.slots(1, lens[1])
    for pos in (3, lens[1] // 2):
        cache.pages(1)[pg[pos], r[pos], 1, 7 + pos % 2] = to_type(np.float32([value]), act)[0]
    cache.upload(mlk)
    cache.handle = paged.PagedCache(cache.k, cache.v, act, batch.n_pages, batch.page, KV, hd)
    q = to_type(rng.standard_normal((batch.T, H, hd)) * (0 if equal else 1), act)
    got = values(run_paged(mlk, paged, batch, cache, q, H, act, workspace=ws), act)
    rows = slice(int(batch.start[1]), int(batch.start[2]))
    hit = np.zeros(got.shape, bool)
    for pos in (3, lens[1] // 2):
        hit[rows, 2:4, 7 + pos % 2] = True
    assert (got[hit] == value).all() and np.isfinite(got[~hit]).all()


@pytest.mark.parametrize("act,ct", [("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("name", list(PLANS))
def test_infinite_scores(mlk, paged, name, act, ct):
    """A score of -infinity is weight 0, one of +infinity makes the head's results
    NaN; of the KV head and the tokens that meet it, no others."""
    H, KV, hd = 8, 2, 128
    counts, lens, ws = PLANS[name]
    rng = np.random.default_rng(71)
    batch = Batch(counts, lens, 16, seed=4)
    cache = Cache(mlk, paged, batch, KV, hd, ct, rng)
    x = rng.standard_normal((batch.T, H, hd))
    x[..., 5] = 1.0
    q = to_type(x, act)
    q64 = values(q, act).astype(np.float64)
    n, c = lens[0], counts[0]
    pg, r = batch.slots(0, n)
    good = [a.copy() for a in cache.host]
    for pos in (n - c // 2 - 1, n // 3):
        for value in (-np.inf, np.inf):
            cache.host = [a.copy() for a in good]
            cache.pages(0)[pg[pos], r[pos], 1, 5] = to_type(np.float32([value]), ct)[0]
            cache.upload(mlk)
            cache.handle = paged.PagedCache(cache.k, cache.v, ct, batch.n_pages, batch.page, KV, hd)
            got = run_paged(mlk, paged, batch, cache, q, H, act, workspace=ws)
            g = values(got, act).reshape(batch.T, KV, H // KV, hd)
            sees = [t for t, s, p in batch.rows() if s == 0 and p >= pos]
            others = [t for t, s, p in batch.rows() if s != 0 or p < pos]
            check_paged(batch, cache, q, got, H, act, rows=set(others[-5:]))
            assert np.isfinite(g[:, 0]).all() and np.isfinite(g[others]).all()
            if value > 0:
                assert np.isnan(g[sees, 1]).all()
                continue
            k, v = cache.gathered(0, n)
            for t in sees[::1 + len(sees) // 6]:
                keep = np.delete(np.arange(n - c + t + 1), pos)
                kk, vv = k[keep][:, 1:], v[keep][:, 1:]
                out, pav, d = exact_rows(q64[t, H // 2:], kk, vv, default_scale(hd))
                vsum = np.repeat(np.abs(vv).sum(0), H // KV, axis=0)
                assert_close(values(got[t, H // 2:], act), out, pav, d, len(keep), vsum, act,
                             f"token {t} without position {pos}")


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("name", list(PLANS))
def test_tiny_rows_and_a_tiny_scale(mlk, paged, name, act, ct):
    """Scores that are nothing beside 1: the mean of V, whatever power of two a row
    of q is scaled by on the way (1e-27 is 2^-90, the scale 2^-66).  |score| <= 64 x
    1e-27 x 10 x 1e-20, so its part of the bound is 0."""
    H, KV, hd = 8, 2, 64
    counts, lens, ws = PLANS[name]
    rng = np.random.default_rng(81)
    batch = Batch(counts, lens, 16, seed=4)
    cache = Cache(mlk, paged, batch, KV, hd, ct, rng)
    size = 1e-7 if act == "f16" else 1e-27
    q = to_type(rng.uniform(0.5, 1, (batch.T, H, hd)) * size, act)
    got = run_paged(mlk, paged, batch, cache, q, H, act, scale=1e-20, workspace=ws)
    for t, s, p in batch.rows():
        if t % 7 and p + 1 < lens[s]:
            continue
        k, v = (a[:p + 1] for a in cache.gathered(s, lens[s]))
        out, pav, _ = exact_rows(np.zeros((H, hd)), k, v, 1.0)
        vsum = np.repeat(np.abs(v).sum(0), H // KV, axis=0)
        assert_close(values(got[t], act), out, pav, 0.0, p + 1, vsum, act, f"token {t}, position {p}")


def test_thousands_of_kv_heads_are_left_unsplit(mlk, paged):
    """256 sequences at 8192 KV heads under bounds that ask for a split whose join
    would take 2^23 workgroups: the call runs without it."""
    H = KV = 8192
    hd, n = 2, 256
    rng = np.random.default_rng(91)
    lens = rng.integers(32, 700, n)
    counts = np.ones(n, int)
    counts[100] = 32
    batch = Batch(counts.tolist(), lens.tolist(), 1024)
    batch.n_pages = 2
    batch.table = (np.arange(n) % 2).astype(np.int32).reshape(n, 1)
    cache = Cache(mlk, paged, batch, KV, hd, "f16", rng, fill=False)
    for i in range(2):
        cache.host[i] = to_type(rng.standard_normal(cache.host[i].shape), "f16")
    cache.upload(mlk)
    cache.handle = paged.PagedCache(cache.k, cache.v, "f16", 2, 1024, KV, hd)
    q = to_type(rng.standard_normal((batch.T, H, hd)), "f16")
    got = run_paged(mlk, paged, batch, cache, q, H, "f16")
    assert (got != 7).any(axis=2).all()
    at = int(batch.start[100])
    check_paged(batch, cache, q, got, H, "f16", rows={0, at + 3, at + 31, batch.T - 1})
