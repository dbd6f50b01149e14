"""The next token of each row of logits on the device: temperature, top-k, top-p
and min-p, from the caller's uniform numbers.  The reference's sampler reads the
logits on the host (src/sampler.cc).

    how = Sampling(temperature=d_t, top_k=d_k, top_p=d_p, min_p=d_m)
    ws = DeviceBuffer(workspace_bytes("f32", n_rows, vocab), np.uint8)
    sample("f32", logits, n_rows, vocab, d_u, d_tokens, how=how, workspace=ws)

Types are "f32", "f16" or "bf16"; buffers are DeviceBuffers or device
addresses (a workspace's address needs workspace_bytes).
include/minilamma_hip.h documents the order, the cuts and the bounds.
"""
from __future__ import annotations

import ctypes as C

from . import _p, _sp, check, lib
from .paged import TYPES, _ws_bytes

_i32, _i64, _vp = C.c_int32, C.c_int64, C.c_void_p


class SamplingStruct(C.Structure):
    """mlk_sampling."""
    _fields_ = [("temperature", _vp), ("top_k", _vp), ("top_p", _vp), ("min_p", _vp)]


lib.mlk_sample.argtypes = [_i32, _vp, _i64, _i64, _i64, C.POINTER(SamplingStruct), _vp, _vp, _vp,
                           _vp, C.c_size_t, _vp, _vp]
lib.mlk_sample.restype = C.c_int
lib.mlk_sample_workspace_bytes.argtypes = [_i32, _i64, _i64]
lib.mlk_sample_workspace_bytes.restype = _i64


class Sampling:
    """How each row's token is chosen: device arrays [n_rows], float32 but for
    top_k's int32; None leaves all as it is (temperature None: 1)."""

    def __init__(self, temperature=None, top_k=None, top_p=None, min_p=None):
        self._keep = (temperature, top_k, top_p, min_p)
        self.struct = SamplingStruct(_p(temperature), _p(top_k), _p(top_p), _p(min_p))


def workspace_bytes(type, n_rows, vocab):
    """Bytes of the workspace of sample()."""
    return int(lib.mlk_sample_workspace_bytes(TYPES[type], n_rows, vocab))


def sample(type, logits, n_rows, vocab, uniform, tokens, how=None, prob=None, row_stride=None,
           workspace=None, workspace_bytes=None, err=None, stream=None):
    """tokens [n_rows] int32: each row's choice from its uniform number; prob
    [n_rows] float32: its share of what was kept.  how None: all tokens at
    temperature 1."""
    check(lib.mlk_sample(
        TYPES[type], _p(logits), vocab if row_stride is None else row_stride, n_rows, vocab,
        None if how is None else C.byref(how.struct), _p(uniform), _p(tokens), _p(prob),
        _p(workspace), _ws_bytes(workspace, workspace_bytes), _p(err), _sp(stream)), "mlk_sample")
