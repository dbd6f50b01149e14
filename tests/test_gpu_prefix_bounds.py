"""Prefix lengths far below zero in device memory: no prefix, as any negative one."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from paged_cases import PAIRS, Batch, to_type
from test_gpu_scored import Masks, Pages, check, run_paged, some_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged(mlk):
    return importlib.import_module(mlk.__name__ + ".paged")


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("prefix", [-2 ** 31, -2 ** 31 + 1])
def test_least_prefix_lengths(mlk, paged, prefix, act, ct):
    """Single tokens, chunks and both, whole and split, with and without a workspace."""
    H, KV, hd = 8, 2, 64
    rng = np.random.default_rng(21)
    for counts, lens, page in (([1, 1, 1], [5, 700, 1500], 16), ([75, 3], [333, 40], 16),
                               ([1, 150, 1], [900, 1700, 64], 32)):
        batch = Batch(counts, lens, page, 2)
        pages = Pages(mlk, paged, batch, KV, hd, ct, rng)
        for kw in (dict(), dict(window=100, cap=20.0)):
            masks = Masks(batch, H, prefix=prefix, **kw)
            q = to_type(rng.standard_normal((batch.T, H, hd)), act)
            for ws in (True, False):
                got = run_paged(mlk, paged, batch, pages, masks, q, H, act, workspace=ws)
                check(batch, pages.of, masks, q, got, H, hd, act, rows=some_rows(rng, batch, H))
