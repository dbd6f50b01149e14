"""The operators of a server's attention as timed cases: many sequences over one paged KV cache.

Three kinds, each through the library's public entry points:

  append  the new tokens' keys and values to their pages, with RoPE on q and k on the way
  paged   attention of the new tokens over the paged cache: one token per sequence (a decode
          step), a chunk of a prompt, or both in one batch
  packed  causal attention of whole prompts of different lengths, packed in one buffer

Activations are fp32 (the library's own) or 16-bit; the cache has the activations' type, or 16 bits
under fp32 activations.  Head layouts are the Llama-3-8B and Llama-3-70B ones, the tiny
configuration of cpp-minilamma_amd/workloads.py, and small ones such as tests/ uses.
"""
from __future__ import annotations

import importlib
import math
import random

import torch

own = False  # true: `run` makes the library's calls; false: the plain form

DEV = "cuda"
SHAPES = {  # n_heads, n_kv_heads, head_dim, theta
    "tiny": (4, 2, 16, 10000.0),
    "8b": (32, 8, 128, 500000.0),
    "70b": (64, 8, 128, 500000.0),
    "small64": (16, 4, 64, 10000.0),
    "multi64": (12, 12, 64, 10000.0),
    "small80": (8, 8, 80, 10000.0),
    "shared256": (8, 1, 256, 10000.0),
}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]

_mods = {}


def _paged():
    """The package's paged-cache module."""
    if not _mods:
        from __graft_entry__ import load_package
        mlk = load_package()
        mlk.set_device(0)
        _mods["paged"] = importlib.import_module(mlk.__name__ + ".paged")
    return _mods["paged"]


# ------------------------------------------------------------------ the cases
# `seqs` sequences; `tokens` new tokens in all, of which `ones` sequences bring one each and the
# others share the rest; `context` is the longest sequence's length after the step.  `mix` picks
# the lengths.

def listed():
    return [
        # the tiny model's first prompt: a launch and its latency
        dict(name="append_tiny_f32_6", kind="append", shape="tiny", act="f32", cache="f32",
             seqs=1, ones=0, tokens=6, context=6, page=16, neox=False, mix=1),
        # a decode step of 64 chats into the half-precision cache of an fp32 server
        dict(name="append_8b_f16_decode_64", kind="append", shape="8b", act="f32", cache="f16",
             seqs=64, ones=64, tokens=64, context=2048, page=16, neox=False, mix=2),
        # five prompts taken in together
        dict(name="append_8b_f16_4096", kind="append", shape="8b", act="f32", cache="f16",
             seqs=5, ones=0, tokens=4096, context=2500, page=16, neox=False, mix=3),
        # a long odd-sized intake at the 70B heads, 16-bit throughout, NeoX pairs
        dict(name="append_70b_bf16_8191", kind="append", shape="70b", act="bf16", cache="bf16",
             seqs=9, ones=2, tokens=8191, context=4096, page=64, neox=True, mix=4),
        # one chat's next token at the end of an 8191-position context, all in fp32
        dict(name="paged_8b_f32_decode_1", kind="paged", shape="8b", act="f32", cache="f32",
             seqs=1, ones=1, tokens=1, context=8191, page=16, mix=5),
        # a decode step of 64 chats of all ages
        dict(name="paged_8b_bf16_decode_64", kind="paged", shape="8b", act="bf16", cache="bf16",
             seqs=64, ones=64, tokens=64, context=8192, page=16, mix=6),
        # four sequences over long documents, 70B heads, fp32 activations on a 16-bit cache
        dict(name="paged_70b_f16_decode_4_long", kind="paged", shape="70b", act="f32",
             cache="f16", seqs=4, ones=4, tokens=4, context=100001, page=64, mix=7),
        # a later, ragged chunk of a chat's prompt
        dict(name="paged_8b_f16_chunk_389", kind="paged", shape="8b", act="f32", cache="f16",
             seqs=1, ones=0, tokens=389, context=1889, page=16, mix=8),
        # a server's mixed step: 30 decoding chats and two prompt chunks
        dict(name="paged_8b_bf16_mixed_1054", kind="paged", shape="8b", act="bf16", cache="bf16",
             seqs=32, ones=30, tokens=1054, context=4096, page=32, mix=9),
        # one short prompt on a small model
        dict(name="packed_small_f16_100", kind="packed", shape="small64", act="f16", cache="f16",
             seqs=1, tokens=100, longest=100, mix=10),
        # nine prompts of an fp32 server
        dict(name="packed_8b_f32_2500", kind="packed", shape="8b", act="f32", cache="f32",
             seqs=9, tokens=2500, longest=900, mix=11),
        # long prompts at the 70B heads
        dict(name="packed_70b_bf16_9001", kind="packed", shape="70b", act="bf16", cache="bf16",
             seqs=3, tokens=9001, longest=5000, mix=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "paged", "paged", "packed"])
    shape = rng.choice(["8b", "8b", "8b", "70b", "70b", "tiny", "small64", "multi64", "small80",
                        "shared256"])
    act, cache = rng.choice(PAIRS)
    mix = rng.randrange(1 << 20)
    if kind == "append":
        tokens = _log_int(rng, 1, 8191)
        seqs = rng.randint(1, min(tokens, 64))
        ones = seqs if tokens == seqs else rng.randint(0, seqs - 1)
        return dict(kind=kind, shape=shape, act=act, cache=cache, seqs=seqs, ones=ones,
                    tokens=tokens, context=tokens - seqs + rng.randint(1, 2000),
                    page=rng.choice([8, 16, 32, 64, 256]), neox=rng.random() < 0.5, mix=mix)
    if kind == "paged":
        what = rng.choice(["decode", "decode", "chunk", "mixed"])
        context = _log_int(rng, 300, 30000)
        if what == "decode":
            seqs = _log_int(rng, 1, max(1, min(100, 200000 // context)))
            ones = tokens = seqs
        elif what == "chunk":
            context = min(context, 12000)
            seqs, ones = rng.randint(1, 3), 0
            tokens = seqs * _log_int(rng, 2, min(500, context // 2))
        else:
            context = min(context, 4096)
            seqs = rng.randint(3, 24)
            ones = seqs - rng.randint(1, 2)
            tokens = ones + (seqs - ones) * _log_int(rng, 2, min(400, context // 2))
        return dict(kind=kind, shape=shape, act=act, cache=cache, seqs=seqs, ones=ones,
                    tokens=tokens, context=context, page=rng.choice([8, 16, 32, 64, 256]), mix=mix)
    tokens = _log_int(rng, 1, 4500 if shape in ("8b", "70b") else 6000)
    seqs = rng.randint(1, max(1, min(12, tokens // 8)))
    return dict(kind=kind, shape=shape, act=act, cache=act, seqs=seqs, tokens=tokens,
                longest=-(-tokens // seqs) if seqs == 1 else
                min(tokens - seqs + 1, 2 * -(-tokens // seqs)), mix=mix)


def _shares(rng, total, parts, most):
    """`parts` positive whole numbers of sum `total`, none over `most`, uneven."""
    got = [1] * parts
    left = total - parts
    got[0] += min(left, most - 1)
    left -= got[0] - 1
    while left:
        i = rng.randrange(parts)
        add = min(left, most - got[i], rng.randint(1, max(1, total // parts)))
        got[i] += add
        left -= add
    rng.shuffle(got)
    return got


def _lengths(case):
    """(new tokens, length after the step) of each sequence."""
    rng = random.Random(case["mix"])
    S = case["seqs"]
    if case["kind"] == "packed":
        n = _shares(rng, case["tokens"], S, case["longest"])
        return n, n
    ones, top = case["ones"], case["context"]
    n = [1] * ones
    if S > ones:
        n += _shares(rng, case["tokens"] - ones, S - ones, top)
    rng.shuffle(n)
    lens = [rng.randint(max(k, top // 40), top) for k in n]
    lens[n.index(max(n))] = top
    return n, lens


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(DEV)
    g.manual_seed(int(seed))
    return g


def _normal(g, shape, dtype, std=1.0):
    x = torch.empty(shape, device=DEV, dtype=torch.float32)
    return x.normal_(0.0, std, generator=g).to(dtype)


def _inputs(case, seed):
    g = _gen(seed)
    H, KV, hd, _ = SHAPES[case["shape"]]
    n, lens = _lengths(case)
    T = sum(n)
    act, ct = TYPES[case["act"]], TYPES[case["cache"]]
    # a projection's output: q, k and v side by side in one row
    qkv = _normal(g, (T, (H + 2 * KV) * hd), act)
    d = {"q": qkv[:, :H * hd], "k": qkv[:, H * hd:(H + KV) * hd], "v": qkv[:, (H + KV) * hd:],
         "start": torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32,
                               device=DEV), "n": n, "lens": lens, "T": T}
    if case["kind"] == "packed":
        return d
    page = case["page"]
    per_seq = -(-max(lens) // page)
    used = [-(-m // page) for m in lens]
    n_pages = sum(used) + 3
    order = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)
    table = torch.zeros((len(n), per_seq), dtype=torch.int32, device=DEV)
    at = 0
    for s, u in enumerate(used):
        table[s, :u] = order[at:at + u]
        at += u
    d.update(seq_len=torch.tensor(lens, dtype=torch.int32, device=DEV), table=table,
             kp=_normal(g, (n_pages, page, KV, hd), ct), vp=_normal(g, (n_pages, page, KV, hd), ct))
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    H, KV, hd, _ = SHAPES[case["shape"]]
    d["case"] = case
    d["out"] = torch.empty((d["T"], H, hd), device=DEV, dtype=TYPES[case["act"]])
    if own:
        paged = _paged()
        if case["kind"] == "packed":
            need = paged.attention_packed_workspace_bytes(
                case["act"], len(d["n"]), d["T"], max(d["n"]), H, KV, hd)
        else:
            d["cache"] = paged.PagedCache(
                d["kp"].data_ptr(), d["vp"].data_ptr(), case["cache"], d["kp"].shape[0],
                case["page"], KV, hd)
            d["batch"] = paged.PagedBatch(
                d["start"].data_ptr(), d["seq_len"].data_ptr(), d["table"].data_ptr(),
                len(d["n"]), d["T"], d["table"].shape[1], max(d["n"]), max(d["lens"]))
            need = 0 if case["kind"] == "append" else \
                paged.attention_workspace_bytes(d["cache"], d["batch"], H, case["act"])
        d["ws"] = torch.empty(max(need, 16), device=DEV, dtype=torch.uint8)
    return d


# ------------------------------------------------------------------ one pass

def _run_own(d):
    paged = _paged()
    case = d["case"]
    H, KV, hd, theta = SHAPES[case["shape"]]
    q, k, v = d["q"], d["k"], d["v"]
    if case["kind"] == "append":
        paged.kv_append(d["cache"], d["batch"], k.data_ptr(), v.data_ptr(), case["act"],
                        q=q.data_ptr(), q_out=d["out"].data_ptr(), n_heads=H, theta=theta,
                        rope_type=1 if case["neox"] else 0, q_row_stride=q.stride(0),
                        k_row_stride=k.stride(0), v_row_stride=v.stride(0))
        return d["out"], d["kp"], d["vp"]
    if case["kind"] == "paged":
        paged.attention(d["cache"], d["batch"], q.data_ptr(), d["out"].data_ptr(), H, case["act"],
                        q_row_stride=q.stride(0), workspace=d["ws"].data_ptr(),
                        workspace_bytes=d["ws"].numel())
        return d["out"]
    paged.attention_packed(case["act"], q.data_ptr(), k.data_ptr(), v.data_ptr(),
                           d["start"].data_ptr(), len(d["n"]), d["T"], max(d["n"]), H, KV, hd,
                           d["out"].data_ptr(), q_row_stride=q.stride(0),
                           k_row_stride=k.stride(0), v_row_stride=v.stride(0),
                           workspace=d["ws"].data_ptr(), workspace_bytes=d["ws"].numel())
    return d["out"]


def _tokens(d):
    """Sequence and position within the sequence's new tokens of every token row."""
    t = torch.arange(d["T"], device=DEV)
    start = d["start"].long()
    s = torch.searchsorted(start, t, right=True) - 1
    return s, t - start[s]


def _rotate(x, cos, sin, neox):
    """RoPE of x [T, heads, hd] (fp32), cos and sin [T, 1, hd / 2]."""
    half = x.shape[-1] // 2
    a, b = (x[..., :half], x[..., half:]) if neox else (x[..., 0::2], x[..., 1::2])
    y0, y1 = a * cos - b * sin, a * sin + b * cos
    return torch.cat([y0, y1], -1) if neox else torch.stack([y0, y1], -1).flatten(-2)


def _attend(q, k, v, pos, scale):
    """q [S, N, H, hd] at positions pos [S, N] over k, v [S, L, KV, hd], all fp32."""
    S, N, H, hd = q.shape
    L, KV = k.shape[1], k.shape[2]
    G = H // KV
    q = q.view(S, N, KV, G, hd).permute(0, 2, 3, 1, 4).reshape(S, KV, G * N, hd)
    k = k.permute(0, 2, 3, 1).contiguous()
    w = torch.matmul(q, k).view(S, KV, G, N, L)
    future = torch.arange(L, device=DEV) > pos[..., None]
    w.mul_(scale).masked_fill_(future[:, None, None], -math.inf)
    w.sub_(w.amax(-1, keepdim=True)).exp_()
    w.div_(w.sum(-1, keepdim=True))
    o = torch.matmul(w.view(S, KV, G * N, L), v.permute(0, 2, 1, 3).contiguous())
    return o.view(S, KV, G, N, hd).permute(0, 3, 1, 2, 4).reshape(S, N, H, hd)


def _run_plain(d):
    case = d["case"]
    H, KV, hd, theta = SHAPES[case["shape"]]
    T, start = d["T"], d["start"].long()
    q = d["q"].float().view(T, H, hd)
    k, v = d["k"].float().view(T, KV, hd), d["v"].float().view(T, KV, hd)
    s, i = _tokens(d)
    count = start[1:] - start[:-1]
    N, scale = max(d["n"]), 1.0 / math.sqrt(hd)
    if case["kind"] == "append":
        pos = d["seq_len"].long()[s] - count[s] + i
        f = theta ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
        a = pos.double()[:, None, None] * f
        cos, sin = torch.cos(a).float(), torch.sin(a).float()
        page = d["table"].long()[s, pos // case["page"]]
        row = pos % case["page"]
        d["kp"][page, row] = _rotate(k, cos, sin, case["neox"]).to(d["kp"].dtype)
        d["vp"][page, row] = v.to(d["vp"].dtype)
        d["out"].copy_(_rotate(q, cos, sin, case["neox"]))
        return d["out"], d["kp"], d["vp"]
    # sequences side by side, each padded to the longest
    n = torch.arange(N, device=DEV)
    at = (start[:-1, None] + n).clamp_max(T - 1)
    if case["kind"] == "paged":
        first = (d["seq_len"].long() - count)[:, None]
        L = d["table"].shape[1] * case["page"]
        ks = d["kp"][d["table"].long()].view(-1, L, KV, hd).float()
        vs = d["vp"][d["table"].long()].view(-1, L, KV, hd).float()
    else:
        first = torch.zeros_like(count)[:, None]
        ks, vs = k[at], v[at]
    o = _attend(q[at], ks, vs, first + n, scale)
    d["out"].copy_(o[s, i])
    return d["out"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ what it cannot do without

def work(case):
    H, KV, hd, _ = SHAPES[case["shape"]]
    n, lens = _lengths(case)
    T = sum(n)
    a, c = SIZE[case["act"]], SIZE[case["cache"]]
    if case["kind"] == "append":
        return {"bytes": T * hd * (2 * a * H + 2 * KV * (a + c)) + 4 * T,
                "flops": 3 * T * (H + KV) * hd}
    rows = sum(lens)
    pairs = sum(k * (m - k) + k * (k + 1) // 2 for k, m in zip(n, lens))
    table = 0 if case["kind"] == "packed" else 4 * sum(-(-m // case["page"]) for m in lens)
    return {"bytes": 2 * a * T * H * hd + 2 * c * rows * KV * hd + table + 8 * len(n),
            "flops": 4 * hd * H * pairs}


# ------------------------------------------------------------------ 64 bits, one sequence at a time

def exact(case, seed):
    d = _inputs(case, seed)
    H, KV, hd, theta = SHAPES[case["shape"]]
    q, out = d["q"].double().view(-1, H, hd), []
    k, v = d["k"].double().view(-1, KV, hd), d["v"].double().view(-1, KV, hd)
    if case["kind"] != "packed":
        kp, vp = d["kp"].double(), d["vp"].double()
    for s, (n, m) in enumerate(zip(d["n"], d["lens"])):
        t0 = sum(d["n"][:s])
        qs, ks, vs = q[t0:t0 + n], k[t0:t0 + n], v[t0:t0 + n]
        pos = torch.arange(m - n, m, device=DEV)
        if case["kind"] == "append":
            turn = pos.double()[:, None] / theta ** (
                torch.arange(hd // 2, device=DEV, dtype=torch.float64) * 2 / hd)
            turn = torch.polar(torch.ones_like(turn), turn)[:, None]

            def rotated(x):
                pairs = x.reshape(n, -1, 2, hd // 2).transpose(2, 3) if case["neox"] else \
                    x.reshape(n, -1, hd // 2, 2)
                y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
                return (y.transpose(2, 3) if case["neox"] else y).reshape(x.shape)

            pages = d["table"][s].long()[pos // case["page"]]
            kp[pages, pos % case["page"]] = rotated(ks)
            vp[pages, pos % case["page"]] = vs
            out.append(rotated(qs))
            continue
        if case["kind"] == "paged":
            pages = d["table"][s].long()[:-(-m // case["page"])]
            ks, vs = (x[pages].reshape(-1, KV, hd)[:m] for x in (kp, vp))
        seen = torch.arange(m, device=DEV)[None] <= pos[:, None]
        o = torch.empty_like(qs)
        for h in range(H):
            sc = qs[:, h] @ ks[:, h // (H // KV)].T.contiguous() / math.sqrt(hd)
            o[:, h] = torch.softmax(sc.where(seen, sc.new_tensor(-math.inf)), -1) \
                @ vs[:, h // (H // KV)].contiguous()
        out.append(o)
    out = torch.cat(out)
    return (out, kp, vp) if case["kind"] == "append" else out
