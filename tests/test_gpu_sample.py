"""The sampler on the GPU against its definition in float64.

A weight of the kernel is a whole number of 2^-42 of the largest, so within 2^-43 of
its own value, and may count as 0 below 2^-44; over V logits the sums C_n are within
V * 2^-43 (C_1 = 1) of their own, and prob = w / C_n within (V + 1) * 2^-42 + half a
step of float32.  A cut or a draw that lies nearer to a border than TOL = (V + 1) *
2^-41 of the sum may go to either side: such rows are compared with the definition's
range of answers, all others with its answer.  Where weights are equal the sums are
whole and nothing is near.
"""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from paged_cases import to_type, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sampling(mlk):
    return importlib.import_module(mlk.__name__ + ".sampling")


def define(x, t, k, p, m, u):
    """(token, prob, whether every comparison is clear) of one row of float64
    logits; token -1: refused."""
    if not t >= 0 or np.isnan([p, m]).any() or (t > 0 and not 0 <= u < 1) or np.isnan(x).any() \
            or x.max() == -np.inf:
        return -1, 0.0, True
    order = np.argsort(-x, kind="stable")
    xs = x[order]
    if t == 0:
        return int(order[0]), 1.0, True
    with np.errstate(invalid="ignore"):
        w = np.where(xs == xs[0], 1.0, np.exp((xs - xs[0]) / max(t, 2.0 ** -14)))
    c = np.cumsum(w)
    V = len(x)
    tol = (V + 1) * 2.0 ** -41
    clear = True

    def near(a, b, where):
        return bool((np.abs(a - b) <= tol * np.maximum(b, 1.0))[where].any())

    differ = np.ones(V, bool)  # places whose weight is not the next one's: where sums are inexact
    nk = min(k, V) if k > 0 else V
    n = nk
    equal = (w == 1.0).all()
    if p < 1:
        bound = p * c[nk - 1]
        n = min(n, int((c[:nk] < bound).sum()) + 1)
        clear &= equal or not near(c, bound, differ)
    if m > 0:
        n = min(n, int((w >= m).sum()))
        clear &= not ((np.abs(w - m) <= 2.0 ** -42) & (w != 1.0)).any()
    n = max(n, 1)
    bound = u * c[n - 1]
    clear &= u == 0 or equal or not near(c, bound, differ)
    j = min(int((c[:n] <= bound).sum()), n - 1)
    return int(order[j]), float(w[j] / c[n - 1]), clear


def settings(rows, **kw):
    base = dict(t=1.0, k=0, p=1.0, m=0.0, u=0.5)
    return [dict(base, **{n: v[i] if isinstance(v, (list, np.ndarray)) else v
                          for n, v in kw.items()}) for i in range(rows)]


def run(mlk, sampling, x, how, act="f32", stride=None, offset=0, prob=True, err=None, only=None):
    """x [rows, V] float32 through the device: (tokens, probs, error flag)."""
    rows, V = x.shape
    stride = V if stride is None else stride
    bits = to_type(x, act)
    whole = np.full(offset + rows * stride, 0, bits.dtype)
    if act != "bf16":
        whole[:] = 99  # what lies between rows is not a logit
    else:
        whole[:] = to_type(np.float32([99]), act)[0]
    for r in range(rows):
        whole[offset + r * stride:offset + r * stride + V] = bits[r]
    up = mlk.DeviceBuffer.from_array
    d = up(whole)
    f = {n: up(np.array([h[n] for h in how], np.int32 if n == "k" else np.float32))
         for n in ("t", "k", "p", "m", "u")}
    given = {n: f[n] if only is None or n in only else None for n in ("t", "k", "p", "m")}
    s = sampling.Sampling(given["t"], given["k"], given["p"], given["m"])
    tokens, pr = up(np.full(rows + 1, -77, np.int32)), up(np.full(rows + 1, -7, np.float32))
    flag = up(np.zeros(1, np.int32))
    ws = mlk.DeviceBuffer(sampling.workspace_bytes(act, rows, V), np.uint8)
    sampling.sample(act, d.offset(offset * bits.itemsize), rows, V, f["u"], tokens, how=s,
                    prob=pr if prob else None, row_stride=stride, workspace=ws, err=flag)
    mlk.synchronize()
    tokens, pr = tokens.download(), pr.download()
    assert tokens[-1] == -77 and pr[-1] == -7, "written past the last row"
    return tokens[:-1], pr[:-1], int(flag.download()[0])


def check(x, how, got, act="f32", need_clear=0.9):
    """Every clear row's token and prob; `need_clear` of the rows have to be."""
    tokens, probs, flag = got
    x = values(to_type(x, act), act).astype(np.float64)
    V = x.shape[1]
    clear = 0
    refused = False
    for r, h in enumerate(how):
        h = {n: h[n] if n == "k" else float(np.float32(h[n])) for n in h}
        token, prob, sure = define(x[r], **h)
        refused |= token < 0
        if not sure:
            assert 0 <= tokens[r] < V and 0 <= probs[r] <= 1
            continue
        clear += 1
        assert tokens[r] == token, (r, h, int(tokens[r]), token)
        assert abs(probs[r] - prob) <= 2.0 ** -24 * prob + (V + 1) * 2.0 ** -42, (r, h)
    assert clear >= need_clear * len(how), f"{clear} of {len(how)} rows are clear"
    assert (flag != 0) == refused


def logits(rng, rows, V, std=2.0):
    x = rng.standard_normal((rows, V)).astype(np.float32) * np.float32(std)
    some = rng.integers(0, V, (rows, min(V, 30)))
    for r in range(rows):
        x[r, some[r]] += 6
    return x


MIX = [dict(), dict(t=0.7, p=0.9), dict(t=0.9, k=50), dict(t=1.2, m=0.05), dict(t=0.0),
       dict(t=0.8, k=200, p=0.95, m=0.02), dict(t=1.5, p=0.98), dict(k=1), dict(p=0.0),
       dict(t=2.0, p=0.3), dict(k=3, p=0.5), dict(m=1.0), dict(m=0.5, p=0.99), dict(t=0.05),
       dict(t=30.0, p=0.7), dict(k=100000, p=0.6), dict(k=2000)]


def mixed(rng, rows=len(MIX)):
    """MIX's settings in turn, each row with a uniform number of its own."""
    return [{**settings(1)[0], **MIX[r % len(MIX)], "u": float(np.float32(rng.random() * (1 - 2.0 ** -24)))}
            for r in range(rows)]


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 131, 1000, 4097, 32000, 50257, 128256, 200003])
def test_sampling(mlk, sampling, V, act):
    rng = np.random.default_rng(V)
    x = logits(rng, len(MIX), V)
    how = mixed(rng)
    check(x, how, run(mlk, sampling, x, how, act), act, 0.8)


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
def test_every_place_of_a_small_row_is_drawn_from_its_share(mlk, sampling, act):
    """u in the middle of each token's share of a row of nine."""
    x = np.float32([[0.5, 3.0, -1.0, 3.0, 2.0, -np.inf, 0.5, 2.5, 1.0]])
    order = np.argsort(-x[0], kind="stable")
    w = np.exp(x[0, order].astype(np.float64) - 3.0)
    c = np.cumsum(w)
    rows = 8
    u = (c[:rows] - w[:rows] / 2) / c[-1]
    how = settings(rows, u=u.astype(np.float32))
    tokens, probs, flag = run(mlk, sampling, np.repeat(x, rows, 0), how, act)
    np.testing.assert_array_equal(tokens, order[:rows])
    np.testing.assert_allclose(probs, w[:rows] / c[-1], rtol=2.0 ** -23)
    assert flag == 0


@pytest.mark.parametrize("V", [7, 1000, 70001])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
def test_equal_logits_go_by_index(mlk, sampling, act, V):
    """All logits equal, at ordinary and at the type's lowest values (a mask that
    leaves none): the first n, of equal shares."""
    lowest = {"f32": np.finfo(np.float32).min, "f16": np.float32(-65504.0),
              "bf16": values(np.uint16([0xFF7F]), "bf16")[0]}[act]
    for value in (0.0, -0.0, 1.5, -3.0, lowest):
        x = np.full((8, V), value, np.float32)
        how = settings(8, u=[0.0, 0.25, 0.5, 1 - 2.0 ** -24, 0.5, 0.25, 0.75, 0.5],
                       k=[0, 0, 0, 0, 3, 0, 2, 0], p=[1, 1, 1, 1, 1, 0.5, 0.5, 1.0],
                       m=[0, 0, 0, 0, 0, 0, 0, 1.0])
        check(x, how, run(mlk, sampling, x, how, act), act, 1.0)
    x[:, ::2], x[:, 1::2] = 0.0, -0.0  # equal too
    check(x, how, run(mlk, sampling, x, how, act), act, 1.0)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("V", [130, 40000, 128256])
def test_ties_in_the_middle(mlk, sampling, act, V):
    """Logits of few values: thousands of equal ones at every cut."""
    rng = np.random.default_rng(V)
    x = rng.integers(-3, 3, (len(MIX), V)).astype(np.float32)
    how = mixed(rng)
    check(x, how, run(mlk, sampling, x, how, act), act, 0.5)


@pytest.mark.parametrize("V", [9, 500, 30000])
def test_cuts_among_equal_largest_logits(mlk, sampling, V):
    """Three equal largest logits: min-p of 1 keeps the three, more than 1 the first, a
    top-k of 2 two, a top-p the fewest that reach it."""
    x = np.zeros((8, V), np.float32)
    x[:, [2, V // 2, V - 2]] = 60.0  # all else weighs nothing
    how = settings(8, m=[1.0, 1.5, 3.0, 1.0, 0, 0, 0, 0], k=[0, 0, 0, 2, 2, 0, 0, 1],
                   p=[1, 1, 1, 1, 1, 0.5, 0.3, 1], u=[0.99, 0.99, 0.5, 0.99, 0.99, 0.99, 0.99, 0.99])
    tokens, probs, flag = run(mlk, sampling, x, how)
    a, b, c = 2, V // 2, V - 2
    np.testing.assert_array_equal(tokens, [c, a, a, b, b, b, a, a])
    np.testing.assert_allclose(probs, [1 / 3, 1, 1, 1 / 2, 1 / 2, 1 / 2, 1, 1], rtol=2.0 ** -23)
    assert flag == 0


def test_uniforms_at_the_ends(mlk, sampling):
    rng = np.random.default_rng(5)
    x = logits(rng, 6, 5000)
    how = settings(6, u=[0.0, 0.0, 0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 2.0 ** -149],
                   k=[0, 40, 0, 40, 1, 0], p=[1, 1, 0.5, 1, 1, 1])
    got = run(mlk, sampling, x, how)
    check(x, how, got, need_clear=0.6)
    np.testing.assert_array_equal(got[0][[0, 1, 2, 4, 5]], x.argmax(1)[[0, 1, 2, 4, 5]])


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
def test_masked_and_infinite_logits(mlk, sampling, act):
    rng = np.random.default_rng(6)
    V = 9000
    x = logits(rng, 9, V)
    x[0, rng.random(V) < 0.9] = -np.inf
    x[1] = -np.inf
    x[1, 4321] = -2.0          # one is left
    x[2] = -np.inf             # none is
    x[3, 17] = np.inf          # takes all
    x[4, [5, 8000]] = np.inf   # share it
    x[5, 100] = np.nan
    x[6, V - 1] = np.nan
    x[7] = -np.inf
    x[7, [3, 8999]] = values(to_type(np.float32([-60000.0]), act), act)[0]
    how = settings(9, u=[0.3, 0.99, 0.5, 0.9, 0.75, 0.5, 0.0, 0.75, 0.5], k=[0, 9, 0, 0, 0, 0, 0, 0, 5],
                   t=[1, 1, 1, 1, 1, 1, 0, 1, 1])
    got = run(mlk, sampling, x, how, act)
    check(x, how, got, act, 1.0)
    np.testing.assert_array_equal(got[0][[1, 2, 3, 4, 5, 6, 7]], [4321, -1, 17, 8000, -1, -1, 8999])


def test_settings_that_cannot_be(mlk, sampling):
    rng = np.random.default_rng(7)
    x = logits(rng, 12, 300)
    nan = float("nan")
    how = settings(12, t=[nan, -1, 1, 1, 1, 1, 1, 0, 1, 1, np.inf, 1],
                   p=[1, 1, nan, 1, 1, 1, 1, 1, -0.5, 7.0, 1, 1],
                   m=[0, 0, 0, nan, 0, 0, 0, 0, 0, -1, 0, 3.0],
                   u=[0.5, 0.5, 0.5, 0.5, nan, 1.0, -0.1, nan, 0.9, 0.3, 0.3, 0.7],
                   k=[0] * 8 + [0, -4, 0, 0])
    tokens, probs, flag = run(mlk, sampling, x, how)
    assert flag != 0
    np.testing.assert_array_equal(tokens[:7], -1)
    np.testing.assert_array_equal(probs[:7], 0)
    assert tokens[7] == x[7].argmax() and tokens[8] == x[8].argmax() and tokens[11] == x[11].argmax()
    # a temperature of infinity: all weights 1, in the order of the logits; float32(0.3) * 300 > 90
    assert tokens[10] == np.argsort(-x[10], kind="stable")[90]


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,offset", [(1, 0), (5, 1), (8, 8), (64, 3)])
def test_row_strides_and_alignment(mlk, sampling, act, pad, offset):
    rng = np.random.default_rng(8)
    for V in (131, 40003):
        x = logits(rng, len(MIX), V)
        how = mixed(rng)
        got = run(mlk, sampling, x, how, act, stride=V + pad, offset=offset)
        check(x, how, got, act, 0.8)


def test_settings_left_out(mlk, sampling):
    rng = np.random.default_rng(9)
    x = logits(rng, 8, 2000)
    u = rng.random(8).astype(np.float32)
    for only, kw in (((), {}), (("k",), dict(k=7)), (("t", "m"), dict(t=0.6, m=0.1)),
                     (("p",), dict(p=0.8))):
        how = settings(8, u=u, **kw)
        check(x, how, run(mlk, sampling, x, how, only=only), need_clear=0.9)
    a = run(mlk, sampling, x, settings(8, u=u), prob=False)
    np.testing.assert_array_equal(a[0], run(mlk, sampling, x, settings(8, u=u))[0])
    assert (a[1] == -7).all()


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_a_rows_choice_does_not_depend_on_the_others(mlk, sampling, act):
    """The same rows alone, in a batch, in another order: the same tokens and bits."""
    rng = np.random.default_rng(10)
    rows = 300
    x = logits(rng, 40, 20001)[rng.integers(0, 40, rows)]
    how = mixed(rng, rows)
    all_t, all_p, _ = run(mlk, sampling, x, how, act)
    for some in ([0], [7, 3], list(range(40, 57)), list(range(rows))[::-1]):
        t, p, _ = run(mlk, sampling, x[some], [how[i] for i in some], act)
        np.testing.assert_array_equal(t, all_t[some])
        np.testing.assert_array_equal(p.view(np.uint32), all_p[some].view(np.uint32))


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_hard_rows_choose_alike_in_large_and_small_batches(mlk, sampling, act):
    """Rows of equal, few, masked and cut-off logits, 30 at a time and all at once: the
    same tokens and bits, those of the definition where it is clear."""
    rng = np.random.default_rng(14)
    V = 20001
    hard = np.stack([
        np.full(V, 1.5, np.float32), np.full(V, -30000.0, np.float32),
        rng.integers(-3, 3, V).astype(np.float32), rng.integers(0, 2, V).astype(np.float32) * 40,
        np.where(rng.random(V) < 0.9, -np.inf, rng.standard_normal(V)).astype(np.float32),
        np.where(np.arange(V) == 17, 0.0, -np.inf).astype(np.float32), np.full(V, -np.inf, np.float32),
        rng.standard_normal(V).astype(np.float32) * 1e-5, logits(rng, 1, V, 0.3)[0],
        rng.standard_normal(V).astype(np.float32) * 1000])
    x = np.repeat(hard, len(MIX), axis=0)
    x = np.concatenate([x, x])
    how = mixed(rng, len(x))
    all_t, all_p, flag = run(mlk, sampling, x, how, act)
    assert flag != 0  # of the rows that have no logit
    for a in range(0, len(x), 30):
        t, p, _ = run(mlk, sampling, x[a:a + 30], how[a:a + 30], act)
        np.testing.assert_array_equal(t, all_t[a:a + 30])
        np.testing.assert_array_equal(p.view(np.uint32), all_p[a:a + 30].view(np.uint32))
    check(x[:170], how[:170], (all_t[:170], all_p[:170], flag), act, 0.3)


@pytest.mark.parametrize("act,rows", [("f32", 220), ("f32", 500), ("bf16", 400), ("bf16", 700)])
def test_batches_of_every_division(mlk, sampling, act, rows):
    """Batches whose rows are gathered by fewer workgroups each: as 20 of them choose."""
    rng = np.random.default_rng(rows)
    V = 50257
    some = logits(rng, 20, V)
    some[3:6] = np.round(some[3:6])
    some[7, 100:] = -np.inf
    how = mixed(rng, 20)
    few_t, few_p, _ = run(mlk, sampling, some, how, act)
    at = rng.integers(0, 20, rows)
    t, p, _ = run(mlk, sampling, some[at], [how[i] for i in at], act)
    np.testing.assert_array_equal(t, few_t[at])
    np.testing.assert_array_equal(p.view(np.uint32), few_p[at].view(np.uint32))
    check(some, how, (few_t, few_p, 0), act, 0.7)


def test_large_and_far_apart_logits(mlk, sampling):
    """Logits of 10^4 and beyond, all far below 0, spread over 10^5 temperatures."""
    rng = np.random.default_rng(11)
    V = 30000
    base = rng.standard_normal((6, V)).astype(np.float32)
    x = np.stack([base[0] + 20000, base[1] - 50000, base[2] * 300, base[3] * 1e-6, base[4] * 30,
                  base[5] * 1000])
    how = settings(6, t=[1.0, 1.0, 1.0, 1.0, 0.01, 100.0], p=[0.9, 1.0, 0.99, 0.5, 1.0, 0.95],
                   u=rng.random(6).astype(np.float32))
    check(x, how, run(mlk, sampling, x, how), need_clear=0.8)


def test_the_largest_vocabulary(mlk, sampling):
    rng = np.random.default_rng(12)
    V = 1 << 20
    x = logits(rng, 4, V, 1.0)
    how = settings(4, p=[0.9, 1.0, 1.0, 1.0], k=[0, 1000, 0, 0], u=rng.random(4).astype(np.float32))
    x[3] = 2.0
    check(x, how, run(mlk, sampling, x, how), need_clear=0.25)


def test_replays_choose_as_calls_do(mlk, sampling):
    rng = np.random.default_rng(13)
    rows, V = 17, 50257
    up = mlk.DeviceBuffer.from_array
    stream = mlk.Stream()
    x, u, tokens = up(logits(rng, rows, V)), up(rng.random(rows).astype(np.float32)), up(np.zeros(rows, np.int32))
    how = sampling.Sampling(up(np.full(rows, 0.8, np.float32)), up(np.full(rows, 60, np.int32)),
                            up(np.full(rows, 0.95, np.float32)))
    ws = mlk.DeviceBuffer(sampling.workspace_bytes("f32", rows, V), np.uint8)

    def call(to, s):
        sampling.sample("f32", x, rows, V, u, to, how=how, workspace=ws, stream=s)

    call(tokens, stream.handle)
    stream.synchronize()
    with mlk.Graph.capture(stream) as g:
        call(tokens, stream.handle)
    for i in range(4):
        x.upload(logits(rng, rows, V))
        u.upload(rng.random(rows).astype(np.float32))
        g.launch()
        stream.synchronize()
        got = tokens.download()
        eager = up(np.zeros(rows, np.int32))
        call(eager, None)
        mlk.synchronize()
        np.testing.assert_array_equal(got, eager.download())


@pytest.mark.parametrize("rows,V", [(1, 128256), (5, 50257), (70, 50257), (300, 9000), (9, 131)])
def test_calls_at_once_over_any_workspace(mlk, sampling, rows, V):
    """Two streams, a workspace each, full of ones: what a call alone chooses."""
    rng = np.random.default_rng(V + rows)
    up = mlk.DeviceBuffer.from_array
    how = mixed(rng, rows)
    x = [logits(rng, rows, V) for _ in range(2)]
    alone = [run(mlk, sampling, a, how) for a in x]
    f = {n: up(np.array([h[n] for h in how], np.int32 if n == "k" else np.float32))
         for n in ("t", "k", "p", "m", "u")}
    s = sampling.Sampling(f["t"], f["k"], f["p"], f["m"])
    need = sampling.workspace_bytes("f32", rows, V)
    streams = [mlk.Stream() for _ in range(2)]
    d = [up(a) for a in x]
    ws = [up(np.full(need, 255, np.uint8)) for _ in range(2)]
    tokens = [[up(np.zeros(rows, np.int32)) for _ in range(8)] for _ in range(2)]
    probs = [[up(np.zeros(rows, np.float32)) for _ in range(8)] for _ in range(2)]
    for i in range(8):
        for j in range(2):
            sampling.sample("f32", d[j], rows, V, f["u"], tokens[j][i], how=s, prob=probs[j][i],
                            workspace=ws[j], stream=streams[j].handle)
    for j in range(2):
        streams[j].synchronize()
        for i in range(8):
            np.testing.assert_array_equal(tokens[j][i].download(), alone[j][0])
            np.testing.assert_array_equal(probs[j][i].download().view(np.uint32), alone[j][1].view(np.uint32))


def test_rows_past_32_bits(mlk, sampling):
    """Rows 3 * 2^29 logits apart."""
    rng = np.random.default_rng(17)
    up = mlk.DeviceBuffer.from_array
    for V in (40003, 1000):
        rows, stride = 4, 3 << 29
        x, how = logits(rng, rows, V), mixed(rng, rows)
        alone = run(mlk, sampling, x, how)
        far = mlk.DeviceBuffer(4 * ((rows - 1) * stride + V), np.uint8)
        for r in range(rows):
            one = np.ascontiguousarray(x[r])
            mlk.check(mlk.lib.mlk_memcpy(far.offset(4 * r * stride), one.ctypes.data, one.nbytes, mlk.H2D))
        f = {n: up(np.array([h[n] for h in how], np.int32 if n == "k" else np.float32))
             for n in ("t", "k", "p", "m", "u")}
        tokens, ws = up(np.zeros(rows, np.int32)), mlk.DeviceBuffer(sampling.workspace_bytes("f32", rows, V), np.uint8)
        sampling.sample("f32", far, rows, V, f["u"], tokens, how=sampling.Sampling(f["t"], f["k"], f["p"], f["m"]),
                        row_stride=stride, workspace=ws)
        mlk.synchronize()
        np.testing.assert_array_equal(tokens.download(), alone[0])
