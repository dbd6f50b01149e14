"""CPU checks of a server's step at its edges: workspace queries without score functions, a
plan without sequences."""
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


@pytest.mark.parametrize("heads", [(32, 8, 128), (64, 8, 128), (8, 2, 64), (8, 1, 256), (12, 12, 64)], ids=str)
def test_workspace_queries_without_scores_are_the_plain_ones(mlk, paged, heads):
    """scores NULL: the bytes that the plain call asks for."""
    lib = mlk.lib
    seen = set()
    for n_seqs, n_tokens, most_new, most_len in (
            (1, 1, 1, 9000), (64, 64, 1, 8192), (1, 300, 300, 5300), (3, 1500, 500, 3300), (20, 900, 450, 30001),
            (3, 152, 150, 4000), (1, 75, 75, 333), (2, 2000, 1000, 1400), (1, 130, 130, 700)):
        plain = lib.mlk_attention_paged_workspace_bytes(n_seqs, n_tokens, most_new, most_len, *heads)
        assert plain == lib.mlk_attention_paged_scored_workspace_bytes(n_seqs, n_tokens, most_new, most_len,
                                                                       *heads, None)
        packed = lib.mlk_attention_packed_workspace_bytes(n_seqs, n_tokens, most_new, *heads)
        assert packed == lib.mlk_attention_packed_scored_workspace_bytes(n_seqs, n_tokens, most_new, *heads, None)
        seen |= {plain, packed}
    assert len(seen) > 3


def test_a_plan_of_no_sequences_checks_where_it_writes(mlk, paged):
    pool = paged.PagePool(FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, 0, 4, 9, 16)
    with pytest.raises(mlk.MlkError, match="token_start"):
        paged.plan(pool, None, 10, 20, 6 * FAKE + 2)
    for taken in range(1, 5):
        with pytest.raises(mlk.MlkError, match="may not alias"):
            paged.plan(pool, None, 10, 20, taken * FAKE)
