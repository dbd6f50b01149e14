"""The sampler on the GPU against the definition's range of answers (sample_ranges.py), for
every row, near a border or not; and rows drawn in the middle of a share, which are clear."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from paged_cases import to_type, values
from sample_ranges import assert_in_range, place_range
from test_gpu_sample import MIX, check, logits, mixed, run, settings

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sampling(mlk):
    return importlib.import_module(mlk.__name__ + ".sampling")


def exact(h):
    return {n: h[n] if n == "k" else float(np.float32(h[n])) for n in h}


def check_ranges(x, how, got, act="f32"):
    """All rows in their range; the mean number of places that was."""
    x = values(to_type(x, act), act).astype(np.float64)
    open_places = []
    for r, h in enumerate(how):
        h = exact(h)
        if h["t"] == 0:
            assert got[0][r] == x[r].argmax()
            continue
        open_places.append(assert_in_range(x[r], h, int(got[0][r]), float(got[1][r]), f"row {r}"))
    return np.mean(open_places)


def kinds(rng, V):
    """name -> logits of len(MIX) rows."""
    n = len(MIX)
    return {
        "spread": logits(rng, n, V),
        "few values": rng.integers(-3, 3, (n, V)).astype(np.float32),
        "flat": rng.standard_normal((n, V)).astype(np.float32) * np.float32(0.5),
        "around 40": (rng.standard_normal((n, V)) * 2 + 40).astype(np.float32),
        "masked": np.where(rng.random((n, V)) < 0.7, -np.inf, rng.standard_normal((n, V)) * 2).astype(np.float32),
    }


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [17, 257, 4097, 40000, 128256])
def test_every_row_is_in_its_range(mlk, sampling, V, act):
    rng = np.random.default_rng(V)
    for name, x in kinds(rng, V).items():
        x[:, V // 2] = 1.0  # (a masked row keeps one)
        how = mixed(rng)
        print(f"{name}, V {V}", flush=True)
        check_ranges(x, how, run(mlk, sampling, x, how, act), act)


def test_every_row_of_the_largest_vocabulary_is_in_its_range(mlk, sampling):
    rng = np.random.default_rng(31)
    V = 1 << 20
    how = mixed(rng)
    for name, x in kinds(rng, V).items():
        x[:, V // 2] = 1.0
        print(name, flush=True)
        check_ranges(x, how, run(mlk, sampling, x, how))


def middle(x, h, rng):
    """Settings like h whose top-p bound and draw lie in the middle of a token's share, of
    tokens that weigh at least 2^-17 of the sum."""
    h = dict(h)
    h.setdefault("u", 0.5)
    x = x.astype(np.float64)
    if h["p"] < 1:
        _, w, c, *_ = place_range(x, **dict(exact(h), p=1.0, m=0.0))
        nk = min(h["k"], len(x)) if h["k"] > 0 else len(x)
        some = np.flatnonzero(w[:nk] >= 2.0 ** -17 * c[nk - 1])
        j = some[len(some) * 3 // 4]
        h["p"] = float(np.float32((c[j] - w[j] / 2) / c[nk - 1]))
    _, w, c, least, most, _, _ = place_range(x, **exact(h))
    assert least == most
    some = np.flatnonzero(w[:most] >= 2.0 ** -17 * c[most - 1])
    j = some[rng.integers(len(some))]
    h["u"] = float(np.float32((c[j] - w[j] / 2) / c[most - 1]))
    return h


def test_draws_in_the_middle_of_a_share(mlk, sampling):
    """Of 2^20 logits, and of vocabularies in use: none near a border, so each has one answer."""
    rng = np.random.default_rng(32)
    for V in (1 << 20, 128256, 40000):
        x = logits(rng, 8, V, 1.0)
        x[4:] += rng.integers(0, 3, (4, V)).astype(np.float32)
        how = settings(8, p=[0.9, 1.0, 1.0, 0.95, 0.5, 1.0, 0.8, 1.0], k=[0, 1000, 0, 200, 0, 20000, 5000, 0],
                       t=[1.0, 1.0, 1.0, 0.8, 1.0, 0.9, 1.0, 0.7])
        how = [middle(x[r], h, rng) for r, h in enumerate(how)]
        check(x, how, run(mlk, sampling, x, how), need_clear=1.0)
