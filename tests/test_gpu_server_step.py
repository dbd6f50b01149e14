"""A server's step on the device alone: page plan, append, attention with scores and
masks, logits, sampling, and the chosen tokens as the next step's input; eager and
as one captured graph, each stage against its definition from the device's inputs."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from paged_cases import default_scale
from scored_cases import assert_within, scored_rows, seen_by
from test_gpu_plan import Pool
from test_gpu_sample import define

pytestmark = pytest.mark.gpu

H, KV, HD, V, D, PAGE, WIDTH = 4, 2, 16, 131, 64, 8, 12
CAP, WINDOW = 10.0, 30


@pytest.fixture(scope="module")
def paged(mlk):
    return importlib.import_module(mlk.__name__ + ".paged")


@pytest.fixture(scope="module")
def sampling(mlk):
    return importlib.import_module(mlk.__name__ + ".sampling")


class Server:
    """One layer without its feed-forward: embedding -> q, k, v -> pages -> attention ->
    projection -> logits -> tokens, for up to n_tokens rows of S sequences."""

    def __init__(self, mlk, paged, sampling, lens, n_tokens, spare, seed=0):
        self.mlk, self.paged, self.sampling = mlk, paged, sampling
        rng = np.random.default_rng(seed)
        self.S, self.T = len(lens), n_tokens
        up = mlk.DeviceBuffer.from_array
        self.pool = Pool(lens, PAGE, WIDTH, spare, seed).upload(mlk, paged)
        normal = lambda *s, std=1.0: (rng.standard_normal(s) * std).astype(np.float32)  # noqa: E731
        self.w = dict(embed=normal(V, D), qkv=normal((H + 2 * KV) * HD, D, std=0.2),
                      out=normal(V, H * HD, std=0.5), bias=normal(H, std=0.1) ** 2)
        self.d = {n: up(a) for n, a in self.w.items()}
        self.kv = [normal(self.pool.n_pages, PAGE, KV, HD) for _ in range(2)]
        self.d_kv = [up(a) for a in self.kv]
        zeros = lambda n, t=np.float32: up(np.zeros(n, t))  # noqa: E731
        self.tokens, self.start = zeros(n_tokens, np.int32), zeros(self.S + 1, np.int32)
        self.new, self.positions = zeros(self.S, np.int32), zeros(n_tokens, np.int32)
        self.slots, self.err = zeros(n_tokens, np.int64), zeros(1, np.int32)
        self.x, self.qkv = zeros((n_tokens, D)), zeros((n_tokens, (H + 2 * KV) * HD))
        self.att, self.logits = zeros((n_tokens, H * HD)), zeros((n_tokens, V))
        self.q = zeros((n_tokens, H * HD))
        self.u, self.prob = zeros(n_tokens), zeros(n_tokens)
        self.chosen = zeros(n_tokens, np.int32)
        self.settings = [up(np.full(n_tokens, v, t)) for v, t in
                         ((0.8, np.float32), (20, np.int32), (0.9, np.float32), (0.01, np.float32))]
        self.how = sampling.Sampling(*self.settings)
        self.ws_sample = mlk.DeviceBuffer(sampling.workspace_bytes("f32", n_tokens, V), np.uint8)
        self.cache = paged.PagedCache(*self.d_kv, "f32", self.pool.n_pages, PAGE, KV, HD)
        self.batch = paged.PagedBatch(self.start, self.pool.dev["len"], self.pool.dev["table"],
                                      self.S, n_tokens, WIDTH, n_tokens, WIDTH * PAGE)
        self.scores = paged.Scores(softcap=CAP, slopes=self.d["bias"], window=WINDOW)
        need = paged.attention_scored_workspace_bytes(self.cache, self.batch, self.scores, H)
        self.ws = mlk.DeviceBuffer(max(need, 16), np.uint8)

    def step(self, stream=None):
        m, p = self.mlk, self.paged
        p.plan(self.pool.handle, self.new, self.T, WIDTH * PAGE, self.start,
               positions=self.positions, slots=self.slots, workspace=self.pool.ws, err=self.err,
               stream=stream)
        m.gather_f32(self.d["embed"], V, D, self.tokens, self.T, self.x, stream=stream)
        m.linear_f32(self.x, self.d["qkv"], self.qkv, self.T, D, (H + 2 * KV) * HD, stream=stream)
        row = (H + 2 * KV) * HD
        p.kv_append(self.cache, self.batch, self.qkv.offset(4 * H * HD),
                    self.qkv.offset(4 * (H + KV) * HD), "f32", q=self.qkv, q_out=self.q, n_heads=H,
                    q_row_stride=row, k_row_stride=row, v_row_stride=row, err=self.err, stream=stream)
        p.attention_scored(self.cache, self.batch, self.scores, self.q, self.att, H, "f32",
                           workspace=self.ws, err=self.err, stream=stream)
        m.linear_f32(self.att, self.d["out"], self.logits, self.T, H * HD, V, stream=stream)
        self.sampling.sample("f32", self.logits, self.T, V, self.u, self.chosen, how=self.how,
                             prob=self.prob, workspace=self.ws_sample, err=self.err, stream=stream)

    def check(self, new, u):
        """The step that has just run, from what it was given."""
        start, rows, _ = self.pool.plan(new, self.T, WIDTH * PAGE)
        self.pool.same("plan")
        np.testing.assert_array_equal(self.start.download(), start)
        n = len(rows)
        np.testing.assert_array_equal(self.positions.download()[:n], [r[0] for r in rows])
        slots = self.slots.download()[:n]
        np.testing.assert_array_equal(slots, [r[2] for r in rows])
        q = self.q.download().reshape(self.T, H, HD).astype(np.float64)
        qkv = self.qkv.download()
        k, v = (b.download().reshape(-1, KV, HD) for b in self.d_kv)
        np.testing.assert_array_equal(v[slots].reshape(n, -1), qkv[:n, (H + KV) * HD:])
        att = self.att.download().reshape(self.T, H, HD)
        for t, (p, s, _) in enumerate(rows):
            m = int(self.pool.len[s])
            j = np.arange(m)
            at = self.pool.table[s, j // PAGE].astype(np.int64) * PAGE + j % PAGE
            out, bound = scored_rows(q[t], k[at].astype(np.float64), v[at].astype(np.float64),
                                     default_scale(HD), p, seen_by(p, m, WINDOW), CAP, self.w["bias"])
            assert_within(att[t], out, bound, f"row {t}")
        logits, chosen = self.logits.download(), self.chosen.download()
        f = lambda x: float(np.float32(x))  # noqa: E731
        clear = 0
        for t in range(n):
            token, prob, sure = define(logits[t].astype(np.float64), f(0.8), 20, f(0.9), f(0.01), float(u[t]))
            if sure:
                clear += 1
                assert chosen[t] == token
        assert clear >= n - 1
        return start, chosen


def test_steps_of_a_server(mlk, paged, sampling):
    rng = np.random.default_rng(1)
    server = Server(mlk, paged, sampling, [0, 9, 40, 16, 0], 24, 20)
    new, tokens = np.array([7, 1, 1, 1, 0], np.int32), rng.integers(0, V, 24).astype(np.int32)
    for i in range(8):
        u = rng.random(24).astype(np.float32)
        server.new.upload(new)
        server.tokens.upload(tokens)
        server.u.upload(u)
        server.step()
        mlk.synchronize()
        start, chosen = server.check(new, u)
        # each sequence goes on with the token of its last row; one ends, one comes in, one
        # speculates three tokens and has two of them rejected
        tokens[:] = 0
        nxt = np.array([1 if start[s + 1] > start[s] else 0 for s in range(5)], np.int32)
        if i == 2:
            keep = np.array([-1, 0, -1, -1, -1], np.int32)
            err = mlk.DeviceBuffer.from_array(np.zeros(1, np.int32))
            paged.release(server.pool.handle, mlk.DeviceBuffer.from_array(keep),
                          workspace=server.pool.ws, err=err)
            server.pool.release(keep)
            server.pool.same("release")
            nxt[1], nxt[4] = 0, 11
        if i == 4:
            nxt[3] = 3
        if i == 5:
            keep = np.array([-1, -1, -1, server.pool.len[3] - 2, -1], np.int32)
            paged.release(server.pool.handle, mlk.DeviceBuffer.from_array(keep), workspace=server.pool.ws)
            server.pool.release(keep)
            server.pool.same("release")
        at = 0
        for s in range(5):
            if nxt[s]:
                tokens[at] = chosen[max(start[s + 1] - 1, 0)]
                at += nxt[s]
        new = nxt
    assert server.err.download()[0] == 0


def test_a_decode_step_as_one_graph(mlk, paged, sampling):
    """Four sequences decode for 20 steps: the graph's choices feed its next replay by one
    copy on the device, beside an eager server with the same numbers."""
    lens = [3, 17, 30, 64]
    a, b = (Server(mlk, paged, sampling, lens, 4, 30, seed=5) for _ in range(2))
    rng = np.random.default_rng(6)
    first = rng.integers(0, V, 4).astype(np.int32)
    for s in (a, b):
        s.new.upload(np.ones(4, np.int32))
        s.tokens.upload(first)
    stream = mlk.Stream()
    a.u.upload(np.zeros(4, np.float32))
    b.u.upload(np.zeros(4, np.float32))
    a.step(stream.handle)  # the first step of both is eager
    b.step()
    stream.synchronize()
    mlk.synchronize()

    def feed(s, st):
        mlk.check(mlk.lib.mlk_memcpy_async(s.tokens.ptr, s.chosen.ptr, 16, mlk.D2D, st))

    feed(a, stream.handle)
    feed(b, None)
    stream.synchronize()
    mlk.synchronize()
    with mlk.Graph.capture(stream) as g:
        a.step(stream.handle)
    a.pool.plan(np.ones(4), 4, WIDTH * PAGE)
    for i in range(20):
        u = rng.random(4).astype(np.float32)
        a.u.upload(u)
        b.u.upload(u)
        g.launch()
        stream.synchronize()
        b.step()
        mlk.synchronize()
        a.check(np.ones(4, np.int32), u)
        for name in ("tokens", "chosen", "start", "positions", "slots"):
            np.testing.assert_array_equal(getattr(a, name).download(), getattr(b, name).download(), name)
        for name in ("att", "logits", "prob"):
            np.testing.assert_array_equal(getattr(a, name).download().view(np.uint32),
                                          getattr(b, name).download().view(np.uint32), name)
        feed(a, stream.handle)
        feed(b, None)
        stream.synchronize()
        mlk.synchronize()
    assert a.err.download()[0] == 0 and b.err.download()[0] == 0
