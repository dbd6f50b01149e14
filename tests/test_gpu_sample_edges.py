"""The sampler at the ends of its ranges: temperatures up to the largest number, infinities
beside logits of any size, bounds that fall exactly on a sum of equal weights, and more rows
than a round of launches takes."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from test_gpu_sample import check, logits, mixed, run, settings

pytestmark = pytest.mark.gpu

LARGEST = float(np.finfo(np.float32).max)


@pytest.fixture(scope="module")
def sampling(mlk):
    return importlib.import_module(mlk.__name__ + ".sampling")


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [300, 5000, 128256])
@pytest.mark.parametrize("t", [1e37, 2e37, 1e38, LARGEST])
def test_a_masked_logit_is_not_chosen_at_the_highest_temperatures(mlk, sampling, t, V, act):
    """Ten logits are left, which weigh the same; cuts that reach past them, few rows and many."""
    rng = np.random.default_rng(V)
    for rows in (12, 290):
        x = np.full((rows, V), -np.inf, np.float32)
        for r in range(rows):
            x[r, rng.choice(V, 10, replace=False)] = rng.standard_normal(10) * 3
        u = np.resize(np.float32([0.05, 0.55, 0.95, 1 - 2.0 ** -24]), rows)
        how = settings(rows, t=t, u=u, k=list(np.resize([40, 0, 40, 7, 20000, 40], rows)),
                       p=list(np.resize([1, 1, 1, 1, 0.93, 0.93, 0.55], rows)),
                       m=list(np.resize([0, 0.1, 0.2, 0, 0], rows)))
        check(x, how, run(mlk, sampling, x, how, act), act, 1.0)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("V", [200, 3000, 5000, 128256])
@pytest.mark.parametrize("t", [1e-30, 2.0 ** -14, 0.01, 1.0, 1e38, LARGEST, float("inf")])
def test_infinities_share_all_the_weight(mlk, sampling, t, V, act):
    """Beside logits of ordinary size, of over 2^24 temperatures and of the largest number."""
    rng = np.random.default_rng(V)
    for rows in (16, 290) if V <= 5000 else (16,):
        x = rng.standard_normal((rows, V)).astype(np.float32)
        n = rng.integers(1, 4, rows)
        for r in range(rows):
            at = rng.choice(V, n[r] + 20, replace=False)
            x[r, at] = [3e38, 60000.0, -np.inf, 2000.0][r % 4]
            x[r, at[:n[r]]] = np.inf
        u = np.resize(np.float32([0.1, 0.4, 0.6, 0.95]), rows)
        how = settings(rows, t=t, u=u, k=list(np.resize([0, 50, 0, 2, 0, 30000, 0], rows)),
                       p=list(np.resize([1, 1, 0.9, 1, 0.6], rows)), m=list(np.resize([0, 0, 0.1], rows)))
        got = run(mlk, sampling, x, how, act)
        # (an infinity over an infinite temperature: as over the largest)
        check(x, [dict(h, t=min(t, LARGEST)) for h in how], got, act, 1.0)


@pytest.mark.parametrize("V", [4098, 50258, 100000, 150000, 1048574])
def test_bounds_that_equal_a_sum(mlk, sampling, V):
    """Equal logits whose weight is an odd whole number: u V and p V are whole, and so is the
    first place behind them (float64's 53 bits do not hold such sums)."""
    for value in (0.1, 1.3, -7.77, 3.14):
        x = np.full((8, V), value, np.float32)
        how = settings(8, u=[0.5, 0.25, 0.75, 0.125, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0.5, 0.5],
                       p=[1, 1, 1, 1, 0.5, 0.25, 0.5, 1], k=[0, 0, 0, 0, 0, 0, 4096, 4094])
        check(x, how, run(mlk, sampling, x, how), need_clear=1.0)


@pytest.mark.parametrize("rows", [3, 300])
def test_bounds_that_equal_a_sum_beside_others(mlk, sampling, rows):
    """n equal logits far above all others: the draw at i / n is the next of them."""
    V = 60000
    n = 50002
    x = np.full((rows, V), -100.0, np.float32)
    x[:, 9000:9000 + n] = 2.3
    how = settings(rows, u=0.5, p=list(np.resize([1.0, 1.0, 0.5], rows)), k=list(np.resize([0, n, 0], rows)))
    tokens, probs, flag = run(mlk, sampling, x, how)
    want = np.resize([9000 + n // 2, 9000 + n // 2, 9000 + n // 4], rows)
    np.testing.assert_array_equal(tokens, want)
    np.testing.assert_allclose(probs, np.resize([1 / n, 1 / n, 2 / n], rows), rtol=2.0 ** -22)
    assert flag == 0


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_more_rows_than_a_round_takes(mlk, sampling, act):
    """2100 rows, more than twice the 1024 that a round of launches works on, and a last round of
    few: as 60 of them choose."""
    rng = np.random.default_rng(41)
    V, rows = 4999, 2100
    x, how = logits(rng, 60, V), mixed(rng, 60)
    few = run(mlk, sampling, x, how, act)
    check(x, how, few, act, 0.7)
    at = rng.integers(0, 60, rows)
    tokens, probs, flag = run(mlk, sampling, x[at], [how[i] for i in at], act, stride=V + 3, offset=1)
    np.testing.assert_array_equal(tokens, few[0][at])
    np.testing.assert_array_equal(probs.view(np.uint32), few[1][at].view(np.uint32))
    assert flag == 0
