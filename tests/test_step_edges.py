"""CPU checks of a server's step at its edges: a plan without sequences."""
from __future__ import annotations

import importlib

import pytest

import __graft_entry__ as entry

FAKE = 4096  # an address that no call below gets to use


@pytest.fixture(scope="module")
def mlk():
    return entry.load_package()


@pytest.fixture(scope="module")
def paged(mlk):
    return importlib.import_module(mlk.__name__ + ".paged")


def test_a_plan_of_no_sequences_checks_where_it_writes(mlk, paged):
    pool = paged.PagePool(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, 0, 4, 9, 16)
    with pytest.raises(mlk.MlkError, match="token_start"):
        paged.plan(pool, None, 10, 20, 6 * FAKE + 2)
    for taken in range(1, 5):
        with pytest.raises(mlk.MlkError, match="may not alias"):
            paged.plan(pool, None, 10, 20, taken * FAKE)
