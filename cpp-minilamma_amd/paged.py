"""Many sequences at once: the pages and token rows of a step, a paged KV cache,
the append of new tokens to it (RoPE on the way), attention of new tokens over
it, and attention of whole prompts packed in one buffer, plain or with score
functions and masks.  The reference keeps one sequence in one contiguous cache
(src/cuda_kvcache.cc) and has no counterpart.

A step of a server:

    cache = PagedCache(k_pages, v_pages, "f16", n_pages, 16, n_kv_heads, head_dim)
    batch = PagedBatch(token_start, seq_len, page_table, n_seqs, n_tokens,
                       table_stride, max_new_tokens, max_seq_len)
    kv_append(cache, batch, k, v, "f32", q=q, q_out=q_rot, n_heads=H, theta=theta)
    attention(cache, batch, q_rot, out, H, "f32", workspace=ws)

where page_table, seq_len and token_start may come from the device's own plan
of the step, new_tokens [n_seqs] on the device:

    pool = PagePool(page_table, seq_len, free_pages, n_free, n_seqs, table_stride,
                    n_pages, 16)
    plan(pool, new_tokens, n_tokens, max_seq_len, token_start, workspace=plan_ws)
    ...
    release(pool, keep, workspace=plan_ws)      # ended or rejected: pages given back

and capped scores, biases by distance, windows, documents and prefixes go
through attention_scored(cache, batch, Scores(softcap=50.0), q_rot, ...).

Types are "f32", "f16" or "bf16"; buffers are DeviceBuffers or device
addresses (a workspace's address needs workspace_bytes).
include/minilamma_hip.h documents layouts and semantics.
"""
from __future__ import annotations

import ctypes as C
import math

from . import ROPE_NORMAL, _p, _sp, check, lib

_i32, _i64, _vp, _f = C.c_int32, C.c_int64, C.c_void_p, C.c_float
TYPES = {"f32": 0, "f16": 1, "bf16": 2}


class CacheStruct(C.Structure):
    """mlk_paged_cache."""
    _fields_ = [("k", _vp), ("v", _vp), ("type", _i32), ("page_size", _i32), ("n_pages", _i64),
                ("page_stride", _i64), ("n_kv_heads", _i32), ("head_dim", _i32)]


class BatchStruct(C.Structure):
    """mlk_paged_batch."""
    _fields_ = [("token_start", _vp), ("seq_len", _vp), ("page_table", _vp), ("n_seqs", _i64),
                ("n_tokens", _i64), ("table_stride", _i64), ("max_new_tokens", _i64),
                ("max_seq_len", _i64)]


class PoolStruct(C.Structure):
    """mlk_paged_pool."""
    _fields_ = [("page_table", _vp), ("seq_len", _vp), ("free_pages", _vp), ("n_free", _vp),
                ("n_seqs", _i64), ("table_stride", _i64), ("n_pages", _i64), ("page_size", _i32)]


class ScoresStruct(C.Structure):
    """mlk_attention_scores."""
    _fields_ = [("softcap", _f), ("slopes", _vp), ("window", _i64), ("prefix_len", _vp),
                ("first", _vp)]


_CB = [C.POINTER(CacheStruct), C.POINTER(BatchStruct)]
lib.mlk_paged_kv_append.argtypes = _CB + [_i32, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _i32,
                                          _f, _i32, _vp, _vp]
lib.mlk_paged_kv_append.restype = C.c_int
lib.mlk_attention_paged.argtypes = _CB + [_i32, _vp, _i64, _vp, _i32, _f, _vp, C.c_size_t, _vp,
                                          _vp]
lib.mlk_attention_paged.restype = C.c_int
lib.mlk_attention_packed.argtypes = [_i32, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64,
                                     _i32, _i32, _i32, _f, _vp, _vp, C.c_size_t, _vp, _vp]
lib.mlk_attention_packed.restype = C.c_int
lib.mlk_attention_paged_workspace_bytes.argtypes = [_i64] * 4 + [_i32] * 3
lib.mlk_attention_paged_workspace_bytes.restype = _i64
lib.mlk_attention_packed_workspace_bytes.argtypes = [_i64] * 3 + [_i32] * 3
lib.mlk_attention_packed_workspace_bytes.restype = _i64

lib.mlk_paged_plan.argtypes = [C.POINTER(PoolStruct), _vp, _i64, _i64, _vp, _vp, _vp, _vp, _vp,
                               C.c_size_t, _vp, _vp]
lib.mlk_paged_plan.restype = C.c_int
lib.mlk_paged_release.argtypes = [C.POINTER(PoolStruct), _vp, _vp, C.c_size_t, _vp, _vp]
lib.mlk_paged_release.restype = C.c_int
lib.mlk_paged_plan_workspace_bytes.argtypes = [_i64]
lib.mlk_paged_plan_workspace_bytes.restype = _i64
lib.mlk_attention_paged_scored.argtypes = _CB + [C.POINTER(ScoresStruct), _i32, _vp, _i64, _vp,
                                                 _i32, _f, _vp, C.c_size_t, _vp, _vp]
lib.mlk_attention_paged_scored.restype = C.c_int
lib.mlk_attention_paged_scored_workspace_bytes.argtypes = [_i64, _i64, _i64, _i64, _i32, _i32,
                                                           _i32, C.POINTER(ScoresStruct)]
lib.mlk_attention_paged_scored_workspace_bytes.restype = _i64
lib.mlk_attention_packed_scored.argtypes = [_i32, C.POINTER(ScoresStruct), _vp, _i64, _vp, _i64,
                                            _vp, _i64, _vp, _i64, _i64, _i64, _i32, _i32, _i32, _f,
                                            _vp, _vp, C.c_size_t, _vp, _vp]
lib.mlk_attention_packed_scored.restype = C.c_int
lib.mlk_attention_packed_scored_workspace_bytes.argtypes = [_i64, _i64, _i64, _i32, _i32, _i32,
                                                            C.POINTER(ScoresStruct)]
lib.mlk_attention_packed_scored_workspace_bytes.restype = _i64


class PagedCache:
    """One layer's key and value pages [n_pages, page_size, n_kv_heads,
    head_dim]; page_stride: elements from one page to the next (None: dense)."""

    def __init__(self, k, v, type, n_pages, page_size, n_kv_heads, head_dim, page_stride=None):
        self._keep = (k, v)
        self.struct = CacheStruct(_p(k), _p(v), TYPES[type], page_size, n_pages,
                                  page_size * n_kv_heads * head_dim if page_stride is None
                                  else page_stride, n_kv_heads, head_dim)


class PagedBatch:
    """The new tokens of n_seqs sequences (device int32 arrays token_start
    [n_seqs + 1], seq_len [n_seqs], page_table [n_seqs, table_stride]) and the
    host's bounds on them."""

    def __init__(self, token_start, seq_len, page_table, n_seqs, n_tokens, table_stride,
                 max_new_tokens, max_seq_len):
        self._keep = (token_start, seq_len, page_table)
        self.struct = BatchStruct(_p(token_start), _p(seq_len), _p(page_table), n_seqs, n_tokens,
                                  table_stride, max_new_tokens, max_seq_len)


def kv_append(cache, batch, k, v, type, q=None, q_out=None, n_heads=0, theta=10000.0,
              rope_type=ROPE_NORMAL, q_row_stride=None, k_row_stride=None, v_row_stride=None,
              q_out_row_stride=None, err=None, stream=None):
    """k, v rows of the batch's new tokens into their pages, k rotated; with q,
    its rotation into q_out (q_out=None: in place).  theta=0: no rotation."""
    c = cache.struct
    row, qrow = c.n_kv_heads * c.head_dim, n_heads * c.head_dim
    qs = qrow if q_row_stride is None else q_row_stride
    if q is not None and q_out is None:
        q_out, q_out_row_stride = q, qs
    check(lib.mlk_paged_kv_append(
        C.byref(c), C.byref(batch.struct), TYPES[type], _p(k),
        row if k_row_stride is None else k_row_stride, _p(v),
        row if v_row_stride is None else v_row_stride, _p(q), qs, _p(q_out),
        qrow if q_out_row_stride is None else q_out_row_stride, n_heads, theta, rope_type,
        _p(err), _sp(stream)), "mlk_paged_kv_append")


def attention_workspace_bytes(cache, batch, n_heads, type="f32"):
    """Bytes of the optional workspace of attention() for these bounds (the
    same for every type)."""
    c, b = cache.struct, batch.struct
    TYPES[type]
    return int(lib.mlk_attention_paged_workspace_bytes(
        b.n_seqs, b.n_tokens, b.max_new_tokens, b.max_seq_len, n_heads, c.n_kv_heads, c.head_dim))


def attention(cache, batch, q, out, n_heads, type, scale=None, q_row_stride=None, workspace=None,
              workspace_bytes=None, err=None, stream=None):
    """out [n_tokens, n_heads, head_dim]: each new token over its sequence's
    positions up to its own; scale None: 1 / sqrt(head_dim)."""
    hd = cache.struct.head_dim
    check(lib.mlk_attention_paged(
        C.byref(cache.struct), C.byref(batch.struct), TYPES[type], _p(q),
        n_heads * hd if q_row_stride is None else q_row_stride, _p(out), n_heads,
        _scale(scale, hd), _p(workspace), _ws_bytes(workspace, workspace_bytes), _p(err),
        _sp(stream)), "mlk_attention_paged")


def attention_packed_workspace_bytes(type, n_seqs, n_tokens, max_seq_len, n_heads, n_kv_heads,
                                     head_dim):
    """Bytes of the optional workspace of attention_packed() (the same for
    every type)."""
    TYPES[type]
    return int(lib.mlk_attention_packed_workspace_bytes(n_seqs, n_tokens, max_seq_len, n_heads,
                                                        n_kv_heads, head_dim))


def attention_packed(type, q, k, v, seq_start, n_seqs, n_tokens, max_seq_len, n_heads, n_kv_heads,
                     head_dim, out, scale=None, q_row_stride=None, k_row_stride=None,
                     v_row_stride=None, workspace=None, workspace_bytes=None, err=None,
                     stream=None):
    """out [n_tokens, n_heads, head_dim]: causal attention within each of the
    n_seqs sequences, rows seq_start[s] .. seq_start[s + 1] - 1."""
    row = n_kv_heads * head_dim
    check(lib.mlk_attention_packed(
        TYPES[type], _p(q), n_heads * head_dim if q_row_stride is None else q_row_stride, _p(k),
        row if k_row_stride is None else k_row_stride, _p(v),
        row if v_row_stride is None else v_row_stride, _p(seq_start), n_seqs, n_tokens,
        max_seq_len, n_heads, n_kv_heads, head_dim, _scale(scale, head_dim), _p(out),
        _p(workspace), _ws_bytes(workspace, workspace_bytes), _p(err), _sp(stream)),
        "mlk_attention_packed")


class PagePool:
    """Who holds which page: device int32 arrays page_table [n_seqs,
    table_stride], seq_len [n_seqs], free_pages [n_pages] (a stack, its top the
    last of n_free [1]), changed in place by plan() and release()."""

    def __init__(self, page_table, seq_len, free_pages, n_free, n_seqs, table_stride, n_pages,
                 page_size):
        self._keep = (page_table, seq_len, free_pages, n_free)
        self.struct = PoolStruct(_p(page_table), _p(seq_len), _p(free_pages), _p(n_free), n_seqs,
                                 table_stride, n_pages, page_size)


def plan_workspace_bytes(pool):
    """Bytes of the workspace of plan() and release()."""
    return int(lib.mlk_paged_plan_workspace_bytes(pool.struct.n_seqs))


def plan(pool, new_tokens, n_tokens, max_seq_len, token_start, positions=None, token_seq=None,
         slots=None, workspace=None, workspace_bytes=None, err=None, stream=None):
    """Pages and rows for new_tokens[s] new tokens of each sequence, first come
    first served; token_start [n_seqs + 1], positions and token_seq [n_tokens]
    int32, slots [n_tokens] int64."""
    check(lib.mlk_paged_plan(C.byref(pool.struct), _p(new_tokens), n_tokens, max_seq_len,
                             _p(token_start), _p(positions), _p(token_seq), _p(slots),
                             _p(workspace), _ws_bytes(workspace, workspace_bytes), _p(err),
                             _sp(stream)), "mlk_paged_plan")


def release(pool, keep, workspace=None, workspace_bytes=None, err=None, stream=None):
    """Each sequence s cut back to keep[s] positions (negative: as it is), its
    other pages given back."""
    check(lib.mlk_paged_release(C.byref(pool.struct), _p(keep), _p(workspace),
                                _ws_bytes(workspace, workspace_bytes), _p(err), _sp(stream)),
          "mlk_paged_release")


class Scores:
    """What scores go through and which positions a token sees: softcap (0: none),
    slopes [n_heads] float32 of a bias by distance, window (0: none), prefix_len
    [n_seqs] and first [n_tokens] int32 (None: none)."""

    def __init__(self, softcap=0.0, slopes=None, window=0, prefix_len=None, first=None):
        self._keep = (slopes, prefix_len, first)
        self.struct = ScoresStruct(softcap, _p(slopes), window, _p(prefix_len), _p(first))


def attention_scored_workspace_bytes(cache, batch, scores, n_heads):
    """Bytes of the optional workspace of attention_scored() for these bounds."""
    c, b = cache.struct, batch.struct
    return int(lib.mlk_attention_paged_scored_workspace_bytes(
        b.n_seqs, b.n_tokens, b.max_new_tokens, b.max_seq_len, n_heads, c.n_kv_heads, c.head_dim,
        C.byref(scores.struct)))


def attention_scored(cache, batch, scores, q, out, n_heads, type, scale=None, q_row_stride=None,
                     workspace=None, workspace_bytes=None, err=None, stream=None):
    """attention() with score functions and masks."""
    hd = cache.struct.head_dim
    check(lib.mlk_attention_paged_scored(
        C.byref(cache.struct), C.byref(batch.struct), C.byref(scores.struct), TYPES[type], _p(q),
        n_heads * hd if q_row_stride is None else q_row_stride, _p(out), n_heads,
        _scale(scale, hd), _p(workspace), _ws_bytes(workspace, workspace_bytes), _p(err),
        _sp(stream)), "mlk_attention_paged_scored")


def attention_packed_scored_workspace_bytes(scores, n_seqs, n_tokens, max_seq_len, n_heads,
                                            n_kv_heads, head_dim):
    """Bytes of the optional workspace of attention_packed_scored()."""
    return int(lib.mlk_attention_packed_scored_workspace_bytes(
        n_seqs, n_tokens, max_seq_len, n_heads, n_kv_heads, head_dim, C.byref(scores.struct)))


def attention_packed_scored(type, scores, q, k, v, seq_start, n_seqs, n_tokens, max_seq_len,
                            n_heads, n_kv_heads, head_dim, out, scale=None, q_row_stride=None,
                            k_row_stride=None, v_row_stride=None, workspace=None,
                            workspace_bytes=None, err=None, stream=None):
    """attention_packed() with score functions and masks."""
    row = n_kv_heads * head_dim
    check(lib.mlk_attention_packed_scored(
        TYPES[type], C.byref(scores.struct), _p(q),
        n_heads * head_dim if q_row_stride is None else q_row_stride, _p(k),
        row if k_row_stride is None else k_row_stride, _p(v),
        row if v_row_stride is None else v_row_stride, _p(seq_start), n_seqs, n_tokens,
        max_seq_len, n_heads, n_kv_heads, head_dim, _scale(scale, head_dim), _p(out),
        _p(workspace), _ws_bytes(workspace, workspace_bytes), _p(err), _sp(stream)),
        "mlk_attention_packed_scored")


def _scale(scale, head_dim):
    return 1.0 / math.sqrt(max(head_dim, 1)) if scale is None else scale


def _ws_bytes(workspace, nbytes):
    if nbytes is not None:
        return nbytes
    if not _p(workspace):
        return 0
    if not hasattr(workspace, "nbytes"):
        raise ValueError("a workspace given as an address needs workspace_bytes")
    return workspace.nbytes
