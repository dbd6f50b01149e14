"""A plan without sequences on the GPU: no token rows, and token_start says so."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged(mlk):
    return importlib.import_module(mlk.__name__ + ".paged")


def test_plan_of_no_sequences(mlk, paged):
    up = mlk.DeviceBuffer.from_array
    table, free = up(np.full(8, -3, np.int32)), up(np.arange(8, dtype=np.int32))
    lens, n_free = up(np.full(4, 5, np.int32)), up(np.full(1, 6, np.int32))
    pool = paged.PagePool(table, lens, free, n_free, 0, 2, 8, 16)
    start = up(np.full(3, 77, np.int32))
    slots, err = up(np.full(4, -9, np.int64)), up(np.zeros(1, np.int32))
    for n_tokens in (0, 4, 1 << 20):
        start.upload(np.full(3, 77, np.int32))
        paged.plan(pool, None, n_tokens, 32, start, slots=slots if n_tokens < 5 else None, err=err)
        mlk.synchronize()
        np.testing.assert_array_equal(start.download(), [0, 77, 77])
    np.testing.assert_array_equal(slots.download(), -9)
    np.testing.assert_array_equal(table.download(), -3)
    np.testing.assert_array_equal(lens.download(), 5)
    np.testing.assert_array_equal(free.download(), np.arange(8))
    assert n_free.download()[0] == 6 and err.download()[0] == 0


def test_plan_of_no_sequences_in_a_graph(mlk, paged):
    """Replayed between steps that leave another count of rows there."""
    up = mlk.DeviceBuffer.from_array
    pool = paged.PagePool(up(np.zeros(8, np.int32)), up(np.zeros(4, np.int32)), up(np.zeros(8, np.int32)),
                          up(np.zeros(1, np.int32)), 0, 2, 8, 16)
    start, stream = up(np.full(1, 77, np.int32)), mlk.Stream()
    paged.plan(pool, None, 4, 32, start, stream=stream.handle)
    stream.synchronize()
    with mlk.Graph.capture(stream) as g:
        paged.plan(pool, None, 4, 32, start, stream=stream.handle)
    for i in range(4):
        start.upload(np.full(1, 100 + i, np.int32))
        g.launch()
        stream.synchronize()
        assert start.download()[0] == 0
