"""The page plan and its release on the GPU against a sequence-by-sequence
restatement; whole numbers, so equal."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged(mlk):
    return importlib.import_module(mlk.__name__ + ".paged")


class Pool:
    """A host pool: sequences of the given lengths on scattered pages, `spare`
    pages free."""

    def __init__(self, lens, page, width, spare, seed=0):
        self.page, self.width = page, width
        self.len = np.asarray(lens, np.int32)
        held = -(-self.len.astype(np.int64) // page)
        self.n_pages = int(held.sum()) + spare
        order = np.random.default_rng(seed).permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(lens), width), -1, np.int32)
        at = 0
        for s, h in enumerate(held):
            self.table[s, :h] = order[at:at + h]
            at += h
        self.free = np.full(self.n_pages, -5, np.int32)
        self.free[:spare] = order[at:]
        self.n_free = np.array([spare], np.int32)

    ARRAYS = ("table", "len", "free", "n_free")

    def upload(self, mlk, paged):
        self.dev = {n: mlk.DeviceBuffer.from_array(getattr(self, n)) for n in self.ARRAYS}
        self.handle = paged.PagePool(*(self.dev[n] for n in self.ARRAYS), len(self.len), self.width,
                                     self.n_pages, self.page)
        self.ws = mlk.DeviceBuffer(max(paged.plan_workspace_bytes(self.handle), 16), np.uint8)
        return self

    def same(self, what=""):
        for n in self.ARRAYS:
            np.testing.assert_array_equal(self.dev[n].download(), getattr(self, n), f"{what} {n}")

    # the definitions, one sequence after the other
    def plan(self, new, n_tokens, max_len):
        P, err = self.page, False
        free = min(max(int(self.n_free[0]), 0), self.n_pages)
        err |= free != int(self.n_free[0])
        pages = asked = popped = 0
        start, rows = [0], []
        for s, n in enumerate(int(x) for x in new):
            m = int(self.len[s])
            if m < 0 or n < 0 or m + n > max_len:
                err = True
                start.append(start[-1])
                continue
            held = -(-m // P)
            need = -(-(m + n) // P) - held
            pages += need
            asked += n
            if (need and pages > free) or asked > n_tokens:
                start.append(start[-1])
                continue
            for j in range(held, held + need):
                popped += 1
                self.table[s, j] = self.free[free - popped]
            for p in range(m, m + n):
                g = int(self.table[s, p // P])
                ok = 0 <= g < self.n_pages
                err |= not ok
                rows.append((p, s, g * P + p % P if ok else -1))
            self.len[s] = m + n
            start.append(start[-1] + n)
        self.n_free[0] = free - popped
        return np.array(start, np.int32), rows, err

    def release(self, keep):
        P, err = self.page, False
        free = min(max(int(self.n_free[0]), 0), self.n_pages)
        err |= free != int(self.n_free[0])
        back = []
        for s, k in enumerate(int(x) for x in keep):
            m = int(self.len[s])
            if k < 0:
                continue
            if k > m or m > self.width * P:
                err = True
                continue
            for j in range(-(-k // P), -(-m // P)):
                back.append(int(self.table[s, j]))
                err |= not 0 <= back[-1] < self.n_pages
                self.table[s, j] = -1
            self.len[s] = k
        total = len(back)
        for i, g in enumerate(back):
            at = free + total - 1 - i
            if at < self.n_pages:
                self.free[at] = g
            else:
                err = True
        self.n_free[0] = min(free + total, self.n_pages)
        return err


def run_plan(mlk, paged, pool, new, n_tokens, max_len, outputs=True, stream=None, bufs=None):
    """The device's plan and the definition's, compared; the device arrays."""
    if bufs is None:
        bufs = plan_buffers(mlk, pool, new, n_tokens)
    rows = bufs[1:4] if outputs else (None, None, None)
    paged.plan(pool.handle, bufs[4], n_tokens, max_len, bufs[0], *rows, workspace=pool.ws,
               err=bufs[5], stream=stream)
    return bufs


def plan_buffers(mlk, pool, new, n_tokens):
    n = max(n_tokens, 1)
    up = mlk.DeviceBuffer.from_array
    return [up(np.full(len(new) + 1, 77, np.int32)), up(np.full(n, -9, np.int32)),
            up(np.full(n, -9, np.int32)), up(np.full(n, -9, np.int64)),
            up(np.asarray(new, np.int32)), up(np.zeros(1, np.int32))]


def check_plan(pool, bufs, new, n_tokens, max_len, outputs=True):
    start, rows, err = pool.plan(new, n_tokens, max_len)
    np.testing.assert_array_equal(bufs[0].download(), start)
    if outputs:
        for i in range(3):
            got = bufs[1 + i].download()
            np.testing.assert_array_equal(got[:len(rows)], [r[i] for r in rows])
            assert (got[len(rows):] == -9).all(), "rows behind the last token were written"
    pool.same("plan")
    assert (bufs[5].download()[0] != 0) == err
    return start


def lengths(rng, n, top):
    return rng.integers(0, top + 1, n)


CASES = {  # lengths, new tokens, page size, spare pages (None: enough), n_tokens (None: all)
    "one": ([0], [1], 16, None, None),
    "first prompt": ([0], [6], 16, None, None),
    "page ends": ([15, 16, 17, 0, 32], [1, 1, 1, 16, 17], 16, None, None),
    "page of one": ([3, 0, 5], [2, 4, 0], 1, None, None),
    "nothing new": ([5, 0, 16], [0, 0, 0], 16, 0, 0),
    "no rows": ([5, 0], [3, 2], 16, None, 0),
    "pages run out": ([16, 3, 16, 16, 30], [1, 1, 1, 20, 1], 16, 1, None),
    "none free": ([16, 3, 0], [1, 1, 1], 16, 0, None),
    "just enough": ([16, 16], [16, 17], 16, 3, None),
    "one short": ([16, 16], [16, 17], 16, 2, None),
    "rows run out": ([4, 4, 4, 4], [5, 6, 0, 1], 8, None, 10),
    "wrong ones": ([-1, 7, 9, 5, 60], [3, -2, 3, 2, 5], 16, None, None),
}


@pytest.mark.parametrize("name", list(CASES))
@pytest.mark.parametrize("outputs", [True, False])
def test_plan(mlk, paged, name, outputs):
    lens, new, page, spare, n_tokens = CASES[name]
    width = 4 if page >= 8 else 9
    need = sum(max(n, 0) for n in new)
    pool = Pool(np.maximum(lens, 0), page, width, need if spare is None else spare)
    pool.len[:] = lens
    pool.upload(mlk, paged)
    T = need if n_tokens is None else n_tokens
    bufs = run_plan(mlk, paged, pool, new, T, width * page, outputs)
    check_plan(pool, bufs, new, T, width * page, outputs)


# n_seqs up to and past what one workgroup scans at once (4096), rows up to and past what
# it works out itself (16384); with many sequences that bring none between
MANY = [(64, 1, 1.0, 300, 16), (1023, 1, 1.0, 900, 16), (4096, 1, 0.5, 100, 32),
        (4097, 1, 1.0, 40, 8), (9000, 3, 0.7, 50, 16), (40, 1200, 0.9, 3000, 64),
        (5000, 400, 0.03, 700, 16), (70000, 1, 0.01, 30, 8), (3, 16384, 0.5, 20000, 256)]


@pytest.mark.parametrize("n,most,share,top,page", MANY)
@pytest.mark.parametrize("short", [False, True])
def test_plan_of_many(mlk, paged, n, most, share, top, page, short):
    rng = np.random.default_rng(n + most)
    new = rng.integers(1, most + 1, n) * (rng.random(n) < share)
    lens = lengths(rng, n, top)
    width = -(-(top + most) // page)
    need = int((-(-(lens + new) // page) - -(-lens // page)).sum())
    pool = Pool(lens, page, width, need * 2 // 3 if short else need + 1, seed=n).upload(mlk, paged)
    T = int(new.sum()) - (int(new[-5:].sum()) if short else 0)
    bufs = run_plan(mlk, paged, pool, new, T, width * page)
    start = check_plan(pool, bufs, new, T, width * page)
    assert short == (start[-1] < new.sum())
    # a step of nothing, then all of it back, but for a third that stays as it is
    keep = np.where(np.arange(n) % 3 == 1, -1, lens).astype(np.int32)
    before = pool.free.copy()
    check_release(mlk, paged, pool, keep)
    assert (pool.free == before).all() or (keep < 0).any()


def check_release(mlk, paged, pool, keep):
    up = mlk.DeviceBuffer.from_array
    d_keep, err = up(np.asarray(keep, np.int32)), up(np.zeros(1, np.int32))
    paged.release(pool.handle, d_keep, workspace=pool.ws, err=err)
    want = pool.release(keep)
    pool.same("release")
    assert (err.download()[0] != 0) == want


def test_a_plan_cut_back_whole_leaves_the_stack_as_it_was(mlk, paged):
    rng = np.random.default_rng(3)
    lens = lengths(rng, 300, 90)
    pool = Pool(lens, 16, 20, 4000).upload(mlk, paged)
    free, table = pool.free.copy(), pool.table.copy()
    new = rng.integers(0, 60, 300)
    bufs = run_plan(mlk, paged, pool, new, int(new.sum()), 320)
    check_plan(pool, bufs, new, int(new.sum()), 320)
    check_release(mlk, paged, pool, lens)
    assert (pool.free == free).all() and (pool.table == table).all()


RELEASE = {  # lengths, keep, page size
    "all": ([5, 16, 17, 0], [0, 0, 0, 0], 16),
    "none": ([5, 16, 17], [-1, -1, -1], 16),
    "same": ([5, 16, 17], [5, 16, 17], 16),
    "rejected tokens": ([18, 33, 16, 40], [17, 30, 15, 33], 16),
    "wrong": ([18, 33, 16], [19, 12, 2 ** 31 - 1], 16),
    "page of one": ([3, 9], [1, 0], 1),
}


@pytest.mark.parametrize("name", list(RELEASE))
def test_release(mlk, paged, name):
    lens, keep, page = RELEASE[name]
    pool = Pool(lens, page, 9, 3).upload(mlk, paged)
    check_release(mlk, paged, pool, keep)


def test_release_of_thousands(mlk, paged):
    rng = np.random.default_rng(8)
    for n, top, page in ((5000, 200, 8), (30, 40000, 16), (4096, 64, 16)):
        lens = lengths(rng, n, top)
        pool = Pool(lens, page, -(-top // page), 7, seed=n).upload(mlk, paged)
        keep = np.where(rng.random(n) < 0.3, 0, np.maximum(lens - rng.integers(0, 9, n), 0))
        keep[rng.random(n) < 0.1] = -1
        check_release(mlk, paged, pool, keep)


def test_pages_and_counts_that_cannot_be(mlk, paged):
    """A free page and a held one outside [0, n_pages), a stack count outside its
    range, a page held twice: raised, and nothing else is harmed."""
    def fresh():
        return Pool([20, 3, 40], 16, 6, 5)
    pool = fresh()
    pool.free[4] = pool.n_pages      # popped first
    pool.table[2, 2] = -3            # where the third's next token goes
    pool.upload(mlk, paged)
    bufs = run_plan(mlk, paged, pool, [15, 1, 2], 18, 96)
    check_plan(pool, bufs, [15, 1, 2], 18, 96)
    assert bufs[5].download()[0] != 0 and (bufs[3].download() == -1).any()
    check_release(mlk, paged, pool, [0, 0, 0])
    for count in (-4, 2 ** 31 - 1):
        pool = fresh()
        pool.n_free[0] = count
        pool.free[:] = np.arange(pool.n_pages)[::-1]
        pool.upload(mlk, paged)
        bufs = run_plan(mlk, paged, pool, [15, 1, 2], 18, 96)
        check_plan(pool, bufs, [15, 1, 2], 18, 96)
    pool = fresh()
    pool.n_free[0] = pool.n_pages - 2  # six pages come back, two fit
    pool.upload(mlk, paged)
    check_release(mlk, paged, pool, [0, 0, 0])


@pytest.mark.parametrize("n", [50, 5000])
def test_plans_in_a_graph(mlk, paged, n):
    """A decode step's plan captured once, replayed as the sequences grow past page
    ends, eager releases between the replays."""
    rng = np.random.default_rng(n)
    lens = lengths(rng, n, 40)
    pool = Pool(lens, 8, 20, 12 * n).upload(mlk, paged)
    new = np.ones(n, np.int32)
    stream = mlk.Stream()
    bufs = plan_buffers(mlk, pool, new, n)
    run_plan(mlk, paged, pool, new, n, 160, stream=stream.handle, bufs=bufs)
    stream.synchronize()
    check_plan(pool, bufs, new, n, 160)
    with mlk.Graph.capture(stream) as g:
        run_plan(mlk, paged, pool, new, n, 160, stream=stream.handle, bufs=bufs)
    for i in range(12):
        g.launch()
        stream.synchronize()
        check_plan(pool, bufs, new, n, 160)
        if i % 4 == 2:
            keep = np.where(rng.random(n) < 0.2, 0, -1)
            check_release(mlk, paged, pool, keep)
