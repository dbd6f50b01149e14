"""CPU checks of the page plan, the scored attention and the sampler: refusals
before any device call, and the masks' index arithmetic compiled for the host."""
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


@pytest.fixture(scope="module")
def sampling(mlk):
    return importlib.import_module(mlk.__name__ + ".sampling")


def pool(paged, **kw):
    a = dict(page_table=FAKE, seq_len=2 * FAKE, free_pages=3 * FAKE, n_free=4 * FAKE, n_seqs=3,
             table_stride=4, n_pages=9, page_size=16)
    return paged.PagePool(**{**a, **kw})


POOL = [
    (dict(page_table=None), "4-byte aligned device arrays"), (dict(n_free=None), "device arrays"),
    (dict(seq_len=FAKE + 2), "4-byte aligned"), (dict(free_pages=FAKE), "must be distinct"),
    (dict(page_size=0), "power of two"), (dict(page_size=24), "power of two"),
    (dict(n_pages=0), "n_pages"), (dict(n_pages=2 ** 30 + 1), "n_pages"),
    (dict(n_seqs=-1), "n_seqs"), (dict(n_seqs=2 ** 20 + 1), "n_seqs"),
    (dict(table_stride=0), "table_stride"),
    (dict(n_seqs=2 ** 20, table_stride=2 ** 11), "fewer than 2\\^31"),
]


@pytest.mark.parametrize("kw,text", POOL, ids=lambda v: str(v)[:40])
def test_pool_refusals(mlk, paged, kw, text):
    ws = dict(workspace=16 * FAKE, workspace_bytes=1 << 30)
    with pytest.raises(mlk.MlkError, match=text):
        paged.plan(pool(paged, **kw), 5 * FAKE, 10, 20, 6 * FAKE, **ws)
    with pytest.raises(mlk.MlkError, match=text):
        paged.release(pool(paged, **kw), 5 * FAKE, **ws)


def test_plan_refusals(mlk, paged):
    ok = dict(pool=pool(paged), new_tokens=5 * FAKE, n_tokens=10, max_seq_len=64,
              token_start=6 * FAKE, positions=7 * FAKE, token_seq=8 * FAKE, slots=9 * FAKE,
              workspace=16 * FAKE, workspace_bytes=64)
    for kw, text in [
            (dict(n_tokens=-1), "n_tokens"), (dict(n_tokens=2 ** 23 + 1), "n_tokens"),
            (dict(max_seq_len=0), "max_seq_len"), (dict(max_seq_len=65), "max_seq_len"),
            (dict(new_tokens=None), "new_tokens"), (dict(token_start=None), "token_start"),
            (dict(positions=FAKE + 2), "4-byte aligned"), (dict(slots=FAKE + 4), "8-byte aligned"),
            (dict(token_seq=7 * FAKE), "may not alias"), (dict(token_start=2 * FAKE), "alias"),
            (dict(slots=5 * FAKE), "may not alias"), (dict(new_tokens=2 * FAKE), "alias seq_len"),
            (dict(workspace=None, workspace_bytes=None), "workspace"),
            (dict(workspace=FAKE + 8), "16-byte"), (dict(workspace_bytes=19), "32 are needed")]:
        with pytest.raises(mlk.MlkError, match=text):
            paged.plan(**{**ok, **kw})
    for kw, text in [
            (dict(keep=None), "keep"), (dict(keep=FAKE + 1), "keep"),
            (dict(keep=2 * FAKE), "may not alias"), (dict(workspace=FAKE + 8), "16-byte"),
            (dict(workspace_bytes=8), "are needed")]:
        args = dict(pool=pool(paged), keep=5 * FAKE, workspace=16 * FAKE, workspace_bytes=64)
        with pytest.raises(mlk.MlkError, match=text):
            paged.release(**{**args, **kw})
    with pytest.raises(mlk.MlkError, match="pool must not be null"):
        mlk.check(mlk.lib.mlk_paged_plan(None, 0, 1, 1, 0, 0, 0, 0, 0, 0, None, None))


def test_plan_of_no_sequences_does_nothing(mlk, paged):
    paged.plan(pool(paged, n_seqs=0), None, 10, 20, None)
    paged.release(pool(paged, n_seqs=0), None)
    assert paged.plan_workspace_bytes(pool(paged, n_seqs=0)) == 0
    assert paged.plan_workspace_bytes(pool(paged, n_seqs=2 ** 20)) >= 4 * 2 ** 20


def make(paged, **kw):
    c = dict(k=FAKE, v=2 * FAKE, type="f16", n_pages=8, page_size=16, n_kv_heads=2, head_dim=8)
    b = dict(token_start=FAKE, seq_len=FAKE, page_table=FAKE, n_seqs=2, n_tokens=4, table_stride=4,
             max_new_tokens=3, max_seq_len=64)
    for name, v in kw.items():
        (b if name in b else c)[name] = v
    return paged.PagedCache(**c), paged.PagedBatch(**b)


SCORES = [
    (dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"),
    (dict(softcap=float("inf")), "softcap"), (dict(window=-1), "window"),
    (dict(softcap=1e-13), "softcap"), (dict(softcap=2e12), "softcap"),
    (dict(slopes=FAKE + 2), "4-byte aligned"), (dict(prefix_len=FAKE + 1), "4-byte aligned"),
    (dict(first=FAKE + 3), "4-byte aligned"), (dict(first=6 * FAKE), "may not alias"),
    (dict(slopes=6 * FAKE), "may not alias"),
]


@pytest.mark.parametrize("kw,text", SCORES, ids=lambda v: str(v)[:40])
def test_scores_refusals(mlk, paged, kw, text):
    cache, batch = make(paged)
    with pytest.raises(mlk.MlkError, match=text):
        paged.attention_scored(cache, batch, paged.Scores(**kw), 5 * FAKE, 6 * FAKE, 4, "f16")
    with pytest.raises(mlk.MlkError, match=text):
        paged.attention_packed_scored("f16", paged.Scores(**kw), 3 * FAKE, 4 * FAKE, 5 * FAKE,
                                      FAKE, 2, 4, 3, 4, 2, 8, 6 * FAKE)


def test_scored_calls_check_the_rest_as_the_plain_ones_do(mlk, paged):
    scores = paged.Scores(softcap=30.0)
    for kw, text in [(dict(page_size=12), "power of two"), (dict(type="bf16"), "own type"),
                     (dict(max_seq_len=65), "exceeds table_stride")]:
        cache, batch = make(paged, **kw)
        with pytest.raises(mlk.MlkError, match="mlk_attention_paged_scored.*" + text):
            paged.attention_scored(cache, batch, scores, 5 * FAKE, 6 * FAKE, 4, "f16")
    cache, batch = make(paged)
    with pytest.raises(mlk.MlkError, match="may not alias q"):
        paged.attention_scored(cache, batch, scores, 5 * FAKE, 5 * FAKE, 4, "f16")
    with pytest.raises(mlk.MlkError, match="mlk_attention_packed_scored.*seq_start"):
        paged.attention_packed_scored("f16", scores, FAKE, 2 * FAKE, 3 * FAKE, None, 2, 4, 3, 4, 2,
                                      8, 6 * FAKE)
    with pytest.raises(ValueError, match="workspace_bytes"):
        paged.attention_scored(cache, batch, scores, 5 * FAKE, 6 * FAKE, 4, "f16", workspace=FAKE)
    with pytest.raises(mlk.MlkError, match="softcap"):  # the scale over it is not a normal number
        paged.attention_scored(cache, batch, scores, 5 * FAKE, 6 * FAKE, 4, "f16", scale=1e-37)
    assert mlk.lib.mlk_attention_packed_scored(0, None, FAKE, 32, FAKE, 16, FAKE, 16, FAKE, 1, 1,
                                               1, 4, 2, 8, 1.0, 9 * FAKE, None, 0, None,
                                               None) == mlk.MLK_ERR_INVALID
    assert b"scores must not be null" in mlk.lib.mlk_last_error()


def test_scored_calls_of_nothing_do_nothing(mlk, paged):
    scores = paged.Scores(softcap=30.0, window=5)
    for kw in (dict(n_seqs=0), dict(n_tokens=0)):
        cache, batch = make(paged, **kw)
        paged.attention_scored(cache, batch, scores, 5 * FAKE, 6 * FAKE, 4, "f16")
        paged.attention_packed_scored("f32", scores, FAKE, 2 * FAKE, 3 * FAKE, None,
                                      kw.get("n_seqs", 2), kw.get("n_tokens", 4), 5, 4, 2, 8,
                                      5 * FAKE)


def test_sample_refusals(mlk, sampling):
    ok = dict(type="f32", logits=FAKE, n_rows=2, vocab=100, uniform=2 * FAKE, tokens=3 * FAKE,
              prob=4 * FAKE, workspace=16 * FAKE, workspace_bytes=1 << 30)
    for kw, text in [
            (dict(logits=None), "logits"), (dict(logits=FAKE + 2), "4-byte aligned"),
            (dict(type="f16", logits=FAKE + 1), "2-byte aligned"),
            (dict(uniform=None), "uniform"), (dict(tokens=None), "tokens"),
            (dict(tokens=FAKE + 2), "4-byte"), (dict(prob=FAKE + 2), "4-byte"),
            (dict(n_rows=-1), "n_rows"), (dict(n_rows=2 ** 20 + 1), "n_rows"),
            (dict(vocab=0), "vocab"), (dict(vocab=2 ** 20 + 1), "vocab"),
            (dict(row_stride=99), "row_stride"), (dict(tokens=FAKE), "may not alias"),
            (dict(prob=2 * FAKE), "may not alias"), (dict(prob=3 * FAKE), "may not alias"),
            (dict(how=sampling.Sampling(top_k=FAKE + 2)), "settings"),
            (dict(how=sampling.Sampling(top_p=3 * FAKE)), "may not alias"),
            (dict(workspace=None, workspace_bytes=None), "workspace"),
            (dict(workspace=FAKE + 8), "16-byte"), (dict(workspace_bytes=8), "workspace")]:
        with pytest.raises(mlk.MlkError, match=text):
            sampling.sample(**{**ok, **kw})
    assert mlk.lib.mlk_sample(3, FAKE, 1, 1, 1, None, FAKE, FAKE, None, None, 0, None,
                              None) == mlk.MLK_ERR_INVALID
    assert b"unknown element type" in mlk.lib.mlk_last_error()
    sampling.sample(**{**ok, "n_rows": 0, "logits": None})
    for bad in ((0, 0, 5), (0, 1, 0), (0, 2 ** 20 + 1, 5), (0, 1, 2 ** 20 + 1), (3, 1, 1)):
        assert mlk.lib.mlk_sample_workspace_bytes(*bad) == 0
    assert sampling.workspace_bytes("f32", 1, 1) > 0


def test_masks_on_the_host(tmp_path):
    """tests/cpp/scored_index.cc: the header the kernels take a token's positions
    from, against the definition, position by position."""
    exe = str(tmp_path / "scored_index")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror",
                    "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "cpp-minilamma_amd", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "scored_index.cc"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
