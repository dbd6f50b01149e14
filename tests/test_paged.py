"""CPU checks of the operators for many sequences: refusals before any device
call, and the kernels' index arithmetic compiled for the host."""
from __future__ import annotations

import importlib
import os
import subprocess

import pytest

import __graft_entry__ as entry

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 4096  # an address that no call below gets to use


@pytest.fixture(scope="module")
def mlk():
    return entry.load_package()


@pytest.fixture(scope="module")
def paged(mlk):
    return importlib.import_module(mlk.__name__ + ".paged")


def make(paged, **kw):
    c = dict(k=FAKE, v=2 * FAKE, type="f16", n_pages=8, page_size=16, n_kv_heads=2, head_dim=8)
    b = dict(token_start=FAKE, seq_len=FAKE, page_table=FAKE, n_seqs=2, n_tokens=4, table_stride=4,
             max_new_tokens=3, max_seq_len=64)
    for name, v in kw.items():
        (b if name in b else c)[name] = v
    return paged.PagedCache(**c), paged.PagedBatch(**b)


SHARED = [
    (dict(k=None), "k pages must not be null"),
    (dict(v=FAKE), "must be distinct"),
    (dict(k=FAKE + 1), "2-byte aligned"),
    (dict(type="bf16"), "cache of their own type"),
    (dict(page_size=12), "power of two"),
    (dict(page_size=0), "power of two"),
    (dict(n_pages=0), "n_pages"),
    (dict(n_pages=2 ** 31), "n_pages"),
    (dict(page_stride=16 * 16 - 1), "page_stride must cover"),
    (dict(n_kv_heads=0), "n_kv_heads"),
    (dict(head_dim=257), "head_dim"),
    (dict(head_dim=0), "head_dim"),
    (dict(n_seqs=-1), "n_seqs"),
    (dict(n_tokens=-1), "n_tokens"),
    (dict(n_tokens=2 ** 28 + 1), "n_tokens"),
    (dict(token_start=None), "must not be null"),
    (dict(seq_len=FAKE + 2), "4-byte aligned"),
    (dict(page_table=None), "must not be null"),
    (dict(table_stride=0), "table_stride"),
    (dict(max_seq_len=65), "exceeds table_stride"),
    (dict(max_seq_len=0), "max_seq_len"),
    (dict(max_new_tokens=0), "max_new_tokens"),
]


@pytest.mark.parametrize("kw,text", SHARED, ids=lambda v: str(v)[:40])
def test_cache_and_batch_refusals(mlk, paged, kw, text):
    cache, batch = make(paged, **kw)
    with pytest.raises(mlk.MlkError, match=text):
        paged.attention(cache, batch, 3 * FAKE, 4 * FAKE, 4, "f16")
    with pytest.raises(mlk.MlkError, match=text):
        paged.kv_append(cache, batch, 3 * FAKE, 4 * FAKE, "f16")


def test_append_refusals(mlk, paged):
    cache, batch = make(paged)
    a, b, q, o = 3 * FAKE, 4 * FAKE, 5 * FAKE, 6 * FAKE
    for args, kw, text in [
            ((None, b), {}, "k must not be null"), ((a, None), {}, "v must not be null"),
            ((a + 1, b), {}, "k must be 2-byte aligned"),
            ((FAKE, b), {}, "may not alias the pages"),
            ((a, b), dict(k_row_stride=15), "row strides"),
            ((a, b), dict(v_row_stride=15), "row strides"),
            ((a, b), dict(theta=-1.0), "theta"), ((a, b), dict(theta=float("nan")), "theta"),
            ((a, b), dict(rope_type=2), "unknown rope type"),
            ((a, b), dict(q=q, q_out=o, n_heads=4, theta=0.0), "q must be null"),
            ((a, b), dict(q=q, q_out=o, n_heads=0), "n_heads"),
            ((a, b), dict(q=q, q_out=o, n_heads=4, q_row_stride=31), "row strides"),
            ((a, b), dict(q=q, q_out=q, n_heads=4, q_row_stride=40), "in place"),
            ((a, b), dict(q=q, q_out=a, n_heads=4), "may not alias"),
            ((a, b), dict(q=q, q_out=FAKE, n_heads=4), "may not alias")]:
        with pytest.raises(mlk.MlkError, match=text):
            paged.kv_append(cache, batch, *args, "f16", **kw)
    odd, batch = make(paged, head_dim=7)
    with pytest.raises(mlk.MlkError, match="even"):
        paged.kv_append(odd, batch, a, b, "f16")


def test_attention_refusals(mlk, paged):
    cache, batch = make(paged)
    q, o = 5 * FAKE, 6 * FAKE
    for args, kw, text in [
            ((None, o, 4), {}, "q must not be null"), ((q, None, 4), {}, "out must not be null"),
            ((q, q, 4), {}, "may not alias"), ((q, FAKE, 4), {}, "may not alias"),
            ((q, o, 3), {}, "multiple of n_kv_heads"), ((q, o, 0), {}, "multiple of n_kv_heads"),
            ((q, o, 4), dict(scale=0.0), "scale"), ((q, o, 4), dict(scale=float("inf")), "scale"),
            ((q, o, 4), dict(q_row_stride=31), "q_row_stride"),
            ((q, o, 4), dict(workspace=FAKE + 4, workspace_bytes=64), "16-byte aligned")]:
        with pytest.raises(mlk.MlkError, match=text):
            paged.attention(cache, batch, *args, "f16", **kw)


def test_packed_refusals(mlk, paged):
    ok = dict(type="f16", q=FAKE, k=2 * FAKE, v=3 * FAKE, seq_start=4 * FAKE, n_seqs=2, n_tokens=9,
              max_seq_len=5, n_heads=4, n_kv_heads=2, head_dim=8, out=5 * FAKE)
    for kw, text in [
            (dict(q=None), "q must not be null"), (dict(out=None), "out must not be null"),
            (dict(k=FAKE * 2 + 1), "k must be 2-byte aligned"), (dict(out=FAKE), "may not alias"),
            (dict(out=3 * FAKE), "may not alias"), (dict(n_heads=3), "multiple of n_kv_heads"),
            (dict(head_dim=300), "head_dim"), (dict(k_row_stride=15), "row strides"),
            (dict(v_row_stride=15), "row strides"), (dict(q_row_stride=31), "row strides"),
            (dict(scale=-1.0), "scale"), (dict(n_seqs=-1), "n_seqs"),
            (dict(n_tokens=2 ** 28 + 1), "n_tokens"), (dict(seq_start=None), "seq_start"),
            (dict(max_seq_len=0), "max_seq_len"),
            (dict(k_row_stride=2 ** 27 + 1), "2\\^27"), (dict(v_row_stride=2 ** 27 + 1), "2\\^27"),
            (dict(n_seqs=2 ** 20, n_tokens=2 ** 20, n_heads=65536, n_kv_heads=65536),
             "workgroups exceed"),
            (dict(workspace=8, workspace_bytes=8), "16-byte aligned")]:
        if "n_kv_heads" in kw:
            kw = dict(kw, k_row_stride=65536 * 8, v_row_stride=65536 * 8)
        with pytest.raises(mlk.MlkError, match=text):
            paged.attention_packed(**{**ok, **kw})


def test_empty_calls_do_nothing(mlk, paged):
    for kw in (dict(n_seqs=0), dict(n_tokens=0)):
        cache, batch = make(paged, **kw)
        paged.attention(cache, batch, 5 * FAKE, 6 * FAKE, 4, "f16")
        paged.kv_append(cache, batch, 3 * FAKE, 4 * FAKE, "f16")
        paged.attention_packed("f32", FAKE, 2 * FAKE, 3 * FAKE, None, kw.get("n_seqs", 2),
                               kw.get("n_tokens", 4), 5, 4, 2, 8, 5 * FAKE)


def test_workspace_bytes_of_bad_and_of_large_bounds(mlk, paged):
    size = mlk.lib.mlk_attention_paged_workspace_bytes
    for bad in ((0, 1, 1, 1, 4, 2, 8), (1, 0, 1, 1, 4, 2, 8), (1, 1, 0, 1, 4, 2, 8),
                (1, 1, 1, 0, 4, 2, 8), (1, 1, 1, 1, 5, 2, 8), (1, 1, 1, 1, 4, 0, 8),
                (1, 1, 1, 1, 4, 2, 257), (2 ** 21, 1, 1, 1, 4, 2, 8)):
        assert size(*bad) == 0
    assert size(1, 1, 1, 100, 32, 8, 128) == 0  # short: nothing is split
    assert 0 < size(64, 64, 1, 131072, 32, 8, 128) < 2 ** 28
    assert size(1, 2 ** 23, 2 ** 23, 2 ** 30, 32, 8, 128) < 2 ** 34
    packed = mlk.lib.mlk_attention_packed_workspace_bytes
    assert packed(3, 100, 2 ** 30, 32, 8, 128) == packed(3, 100, 100, 32, 8, 128)


def test_unknown_types_through_the_c_abi(mlk):
    assert mlk.lib.mlk_attention_packed(3, FAKE, 32, FAKE, 16, FAKE, 16, FAKE, 1, 1, 1, 4, 2, 8,
                                        1.0, FAKE, None, 0, None, None) == mlk.MLK_ERR_INVALID
    assert b"unknown element type" in mlk.lib.mlk_last_error()
    assert mlk.lib.mlk_attention_paged(None, None, 0, None, 0, None, 1, 1.0, None, 0, None,
                                       None) == mlk.MLK_ERR_INVALID


def test_index_arithmetic_on_the_host(tmp_path):
    """tests/cpp/paged_index.cc: the header the kernels take their indexes from,
    over random and wrong sequences and pages."""
    exe = str(tmp_path / "paged_index")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "cpp-minilamma_amd", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "paged_index.cc"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr


def test_many_sequences_are_not_split_beyond_a_launch(mlk, paged):
    """300000 decode tokens and a chunk of 100 at 8 KV heads: 300000 + 100 * 8 /
    256 row tiles and more, times 8, are under 2^22 workgroups and twice that is
    not, so the tile kernel's positions are not split; the few-row partials alone
    remain (2 parts of 512 workgroups at most, 8 heads, 16 rows)."""
    size = mlk.lib.mlk_attention_paged_workspace_bytes
    assert 0 < size(300000, 300100, 100, 8192, 64, 8, 128) <= 2 * 512 * 8 * 16 * (128 * 4 + 8) + 512


def test_bounds_on_counts_are_those_documented(mlk, paged):
    """One more than 2^23 tokens or 2^20 sequences, through every entry."""
    for kw in (dict(n_tokens=2 ** 23 + 1), dict(n_seqs=2 ** 20 + 1)):
        cache, batch = make(paged, **kw)
        with pytest.raises(mlk.MlkError, match="n_seqs must be"):
            paged.attention(cache, batch, 3 * FAKE, 4 * FAKE, 4, "f16")
        with pytest.raises(mlk.MlkError, match="n_seqs must be"):
            paged.kv_append(cache, batch, 3 * FAKE, 4 * FAKE, "f16")
        with pytest.raises(mlk.MlkError, match="n_seqs must be"):
            paged.attention_packed("f16", FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, kw.get("n_seqs", 1),
                                   kw.get("n_tokens", 1), 5, 4, 2, 8, 5 * FAKE)


def test_a_workspace_address_needs_its_size(mlk, paged):
    """A workspace given as an address has no size of its own: without
    workspace_bytes it would go unused."""
    cache, batch = make(paged, n_seqs=0)
    for kw in (dict(workspace=16 * FAKE), dict(workspace=16 * FAKE, workspace_bytes=None)):
        with pytest.raises(ValueError, match="workspace_bytes"):
            paged.attention(cache, batch, 3 * FAKE, 4 * FAKE, 4, "f16", **kw)
        with pytest.raises(ValueError, match="workspace_bytes"):
            paged.attention_packed("f16", FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, 0, 1, 5, 4, 2, 8,
                                   5 * FAKE, **kw)
    paged.attention(cache, batch, 3 * FAKE, 4 * FAKE, 4, "f16", workspace=16 * FAKE,
                    workspace_bytes=0)
    paged.attention(cache, batch, 3 * FAKE, 4 * FAKE, 4, "f16")
