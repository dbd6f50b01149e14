"""What stands around a server's attention as timed cases: a step's page plan, attention with
score functions and masks, and the choice of the next token.

Kinds, each through the library's public entry points:

  step    page table, token rows and cache slots of the new tokens from the requests' lengths, and
          the pages given back (speculated tokens that were all rejected)
  paged   attention over the paged cache with capped scores, a bias by distance, a window, documents
          and prefixes: one token per sequence, chunks of prompts, or both
  packed  the same over whole prompts packed in one buffer
  sample  the next token of every row of logits: temperature, top-k, top-p, min-p, from given
          uniform numbers

Head layouts and vocabularies are those of cpp-minilamma_amd/workloads.py and generic ones such as
tests/ uses.
"""
from __future__ import annotations

import importlib
import math
import random

import torch

own = False  # true: `run` makes the library's calls; false: the plain form

DEV = "cuda"
SHAPES = {  # n_heads, n_kv_heads, head_dim
    "tiny": (4, 2, 16),
    "8b": (32, 8, 128),
    "70b": (64, 8, 128),
    "small64": (16, 4, 64),
    "multi64": (12, 12, 64),
    "small80": (8, 8, 80),
    "shared256": (8, 1, 256),
}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]
VOCABS = [131, 1009, 32000, 50257, 128256]

_mods = {}


def _module(name):
    """One of the package's modules."""
    if name not in _mods:
        from __graft_entry__ import load_package
        mlk = load_package()
        mlk.set_device(0)
        _mods[name] = importlib.import_module(mlk.__name__ + "." + name)
    return _mods[name]


# ------------------------------------------------------------------ the cases
# step, paged and packed: `seqs` sequences, `tokens` new tokens in all, of which `ones` sequences
# bring one each and the others share the rest; `context` is the longest length after the step;
# `mix` picks the lengths.  Score functions: `cap` (0: none), `bias` (by distance), `window` (0:
# none), `docs` (documents within a sequence), `prefix` (a part that sees all of itself).

def listed():
    return [
        # one chat's first prompt on a small server: a launch and its latency
        dict(name="step_6", kind="step", seqs=1, ones=0, tokens=6, context=6, page=16, short=False,
             mix=1),
        # a server's mixed step, 250 chats decode and six prompts come in; pages run out
        dict(name="step_mixed_8186", kind="step", seqs=256, ones=250, tokens=8186, context=9000,
             page=16, short=True, mix=2),
        # the largest intake: prompts of thousands of requests at once
        dict(name="step_262144", kind="step", seqs=4096, ones=1000, tokens=262144, context=20000,
             page=64, short=False, mix=3),
        # one chat's next token with a bias by distance, in fp32
        dict(name="paged_8b_f32_bias_1", kind="paged", shape="8b", act="f32", cache="f32", seqs=1,
             ones=1, tokens=1, context=8191, page=16, cap=0.0, bias=True, window=0, docs=False,
             prefix=False, mix=4),
        # a decode step of 64 chats, capped scores
        dict(name="paged_8b_bf16_cap_64", kind="paged", shape="8b", act="bf16", cache="bf16",
             seqs=64, ones=64, tokens=64, context=8192, page=16, cap=50.0, bias=False, window=0,
             docs=False, prefix=False, mix=5),
        # decode and two prompt chunks at a window of 1000 positions, capped
        dict(name="paged_8b_f16_window_mixed", kind="paged", shape="8b", act="f32", cache="f16",
             seqs=20, ones=18, tokens=900, context=30001, page=32, cap=30.0, bias=False,
             window=1000, docs=False, prefix=False, mix=6),
        # one short prompt of a small model, its head a prefix
        dict(name="packed_small_f16_prefix", kind="packed", shape="small64", act="f16",
             cache="f16", seqs=1, tokens=100, longest=100, cap=0.0, bias=False, window=0,
             docs=False, prefix=True, mix=7),
        # long prompts made of documents, 70B heads, capped
        dict(name="packed_70b_bf16_docs", kind="packed", shape="70b", act="bf16", cache="bf16",
             seqs=3, tokens=7001, longest=4000, cap=50.0, bias=False, window=0, docs=True,
             prefix=False, mix=8),
        # six rows of the tiny model's logits
        dict(name="sample_tiny_f32_6", kind="sample", act="f32", rows=6, vocab=131, how="mixed",
             mix=9),
        # one chat's next token
        dict(name="sample_f32_1", kind="sample", act="f32", rows=1, vocab=128256, how="top_p",
             mix=10),
        # a decode step of 64 chats, each with its own settings
        dict(name="sample_bf16_64", kind="sample", act="bf16", rows=64, vocab=128256, how="mixed",
             mix=11),
        # a large batch
        dict(name="sample_f32_512", kind="sample", act="f32", rows=512, vocab=128256, how="mixed",
             mix=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "paged", "paged", "packed", "packed", "sample", "sample"])
    mix = rng.randrange(1 << 20)
    if kind == "step":
        tokens = _log_int(rng, 1, 200000)
        seqs = min(tokens, _log_int(rng, 1, 4096))
        ones = seqs if tokens == seqs else rng.randint(0, seqs - 1)
        return dict(kind=kind, seqs=seqs, ones=ones, tokens=tokens,
                    context=-(-tokens // max(1, seqs - ones)) * 2 + rng.randint(1, 8000),
                    page=rng.choice([8, 16, 32, 64, 256]), short=rng.random() < 0.4, mix=mix)
    if kind == "sample":
        vocab = rng.choice(VOCABS + [rng.randint(300, 150000)])
        return dict(kind=kind, act=rng.choice(["f32", "f32", "f16", "bf16"]),
                    rows=_log_int(rng, 1, min(2048, 256 * 128256 // vocab)), vocab=vocab,
                    how=rng.choice(["mixed", "mixed", "plain", "top_k", "top_p", "min_p",
                                    "greedy"]), mix=mix)
    shape = rng.choice(["8b", "8b", "8b", "70b", "70b", "tiny", "small64", "multi64", "small80",
                        "shared256"])
    act, cache = rng.choice(PAIRS)
    score = dict(cap=rng.choice([0.0, 0.0, 20.0, 30.0, 50.0]), bias=rng.random() < 0.3,
                 window=rng.choice([0, 0, _log_int(rng, 16, 5000)]), docs=rng.random() < 0.25,
                 prefix=rng.random() < 0.25)
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
                    tokens=tokens, context=context, page=rng.choice([8, 16, 32, 64, 256]),
                    mix=mix, **score)
    tokens = _log_int(rng, 1, 4000 if shape in ("8b", "70b") else 5000)
    seqs = rng.randint(1, max(1, min(12, tokens // 8)))
    return dict(kind=kind, shape=shape, act=act, cache=act, seqs=seqs, tokens=tokens,
                longest=-(-tokens // seqs) if seqs == 1 else
                min(tokens - seqs + 1, 2 * -(-tokens // seqs)), mix=mix, **score)


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


def _masks(case, n, lens):
    """Length of each sequence's prefix (or None) and, for each new token, the first position of
    its document (or None)."""
    rng = random.Random(case["mix"] + 1)
    prefix = [rng.randint(0, m) for m in lens] if case["prefix"] else None
    if not case["docs"]:
        return prefix, None
    first = []
    for k, m in zip(n, lens):
        cuts, at = [], 0
        while at < m:
            cuts.append(at)
            at += rng.randint(max(1, m // 8), max(1, m // 2))
        i = len(cuts) - 1
        row = []
        for p in range(m - 1, m - k - 1, -1):
            while cuts[i] > p:
                i -= 1
            row.append(cuts[i])
        first += row[::-1]
    return prefix, first


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(DEV)
    g.manual_seed(int(seed))
    return g


def _normal(g, shape, dtype, std=1.0):
    x = torch.empty(shape, device=DEV, dtype=torch.float32)
    return x.normal_(0.0, std, generator=g).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _step_inputs(case, seed):
    n, lens = _lengths(case)
    g, page = _gen(seed), case["page"]
    held = [-(-(m - k) // page) for k, m in zip(n, lens)]
    need = [-(-m // page) - h for m, h in zip(lens, held)]
    width = -(-case["context"] // page)
    spare = sum(need) * 9 // 10 if case["short"] else sum(need) + 5
    n_pages = sum(held) + spare
    order = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)
    col = torch.arange(width, device=DEV)
    h = torch.tensor(held, device=DEV)
    at = (torch.cumsum(h, 0) - h)[:, None] + col
    table = torch.where(col < h[:, None], order[at.clamp_max(n_pages - 1)], -1)
    free = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
    free[:spare] = order[sum(held):]
    T = sum(n)
    return {"len": _ints([m - k for k, m in zip(n, lens)]), "new": _ints(n), "T": T,
            "table": table.to(torch.int32).contiguous(), "free": free, "n_free": _ints([spare]),
            "keep": _ints([m - k for k, m in zip(n, lens)]), "pages": n_pages}


def _attention_inputs(case, seed):
    g = _gen(seed)
    H, KV, hd = SHAPES[case["shape"]]
    n, lens = _lengths(case)
    T = sum(n)
    act, ct = TYPES[case["act"]], TYPES[case["cache"]]
    # a projection's output: q, k and v side by side in one row; q as wide as capped scores need
    qkv = _normal(g, (T, (H + 2 * KV) * hd), act, 2.0 if case["cap"] else 1.0)
    prefix, first = _masks(case, n, lens)
    d = {"q": qkv[:, :H * hd], "k": qkv[:, H * hd:(H + KV) * hd], "v": qkv[:, (H + KV) * hd:],
         "start": _ints([sum(n[:i]) for i in range(len(n) + 1)]), "n": n, "lens": lens, "T": T,
         "prefix": None if prefix is None else _ints(prefix),
         "first": None if first is None else _ints(first),
         "slopes": torch.exp2(-8.0 * torch.arange(1, H + 1, device=DEV) / H)
         if case["bias"] else None}
    if case["kind"] == "packed":
        return d
    page = case["page"]
    used = [-(-m // page) for m in lens]
    n_pages = sum(used) + 3
    order = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)
    table = torch.zeros((len(n), -(-max(lens) // page)), dtype=torch.int32, device=DEV)
    at = 0
    for s, u in enumerate(used):
        table[s, :u] = order[at:at + u]
        at += u
    d.update(seq_len=_ints(lens), table=table, kp=_normal(g, (n_pages, page, KV, hd), ct),
             vp=_normal(g, (n_pages, page, KV, hd), ct))
    return d


# temperature, top_k, top_p, min_p of a row
HOW = {
    "plain": (1.0, 0, 1.0, 0.0), "top_k": (0.9, 50, 1.0, 0.0), "top_p": (0.7, 0, 0.9, 0.0),
    "min_p": (1.2, 0, 1.0, 0.05), "greedy": (0.0, 0, 1.0, 0.0), "all": (0.8, 200, 0.95, 0.02),
    "wide": (1.5, 0, 0.98, 0.0),
}


def _sample_inputs(case, seed):
    g, rng = _gen(seed), random.Random(case["mix"])
    R, V = case["rows"], case["vocab"]
    x = _normal(g, (R, V), torch.float32, 2.0)
    # the few that the model favours, and in a third of the rows a grammar that allows 60 %
    likely = torch.randint(V, (R, 40), device=DEV, generator=g)
    x.scatter_add_(1, likely, _normal(g, (R, 40), torch.float32, 2.0) + 6.0)
    banned = torch.rand((R, V), device=DEV, generator=g) < 0.4
    banned[torch.arange(R, device=DEV) % 3 != 2] = False
    x.masked_fill_(banned, -math.inf)
    names = sorted(HOW)
    rows = [HOW[rng.choice(names) if case["how"] == "mixed" else case["how"]] for _ in range(R)]
    t, k, p, m = zip(*rows)
    return {"x": x.to(TYPES[case["act"]]), "u": torch.rand(R, device=DEV, generator=g),
            "t": torch.tensor(t, device=DEV), "k": _ints(k), "p": torch.tensor(p, device=DEV),
            "m": torch.tensor(m, device=DEV)}


def prepare(case, seed):
    if case["kind"] == "step":
        d = _step_inputs(case, seed)
        d["out"] = [torch.zeros(n, dtype=t, device=DEV) for n, t in (
            (case["seqs"] + 1, torch.int32), (d["T"], torch.int32), (d["T"], torch.int32),
            (d["T"], torch.int64))]
    elif case["kind"] == "sample":
        d = _sample_inputs(case, seed)
        d["tokens"] = torch.empty(case["rows"], dtype=torch.int32, device=DEV)
        d["prob"] = torch.empty(case["rows"], dtype=torch.float32, device=DEV)
    else:
        d = _attention_inputs(case, seed)
        H, _, hd = SHAPES[case["shape"]]
        d["out"] = torch.empty((d["T"], H, hd), device=DEV, dtype=TYPES[case["act"]])
    d["case"] = case
    if own:
        _handles(d)
    return d


def _ptr(x):
    return None if x is None else x.data_ptr()


def _handles(d):
    """The handles and the workspace that a program keeps."""
    case = d["case"]
    if case["kind"] == "sample":
        sampling = _module("sampling")
        d["how"] = sampling.Sampling(_ptr(d["t"]), _ptr(d["k"]), _ptr(d["p"]), _ptr(d["m"]))
        need = sampling.workspace_bytes(case["act"], case["rows"], case["vocab"])
    elif case["kind"] == "step":
        paged = _module("paged")
        d["pool"] = paged.PagePool(_ptr(d["table"]), _ptr(d["len"]), _ptr(d["free"]),
                                   _ptr(d["n_free"]), case["seqs"], d["table"].shape[1],
                                   d["pages"], case["page"])
        need = paged.plan_workspace_bytes(d["pool"])
    else:
        paged = _module("paged")
        H, KV, hd = SHAPES[case["shape"]]
        d["scores"] = paged.Scores(softcap=case["cap"], slopes=_ptr(d["slopes"]),
                                   window=case["window"], prefix_len=_ptr(d["prefix"]),
                                   first=_ptr(d["first"]))
        if case["kind"] == "packed":
            need = paged.attention_packed_scored_workspace_bytes(
                d["scores"], len(d["n"]), d["T"], max(d["n"]), H, KV, hd)
        else:
            d["cache"] = paged.PagedCache(_ptr(d["kp"]), _ptr(d["vp"]), case["cache"],
                                          d["kp"].shape[0], case["page"], KV, hd)
            d["batch"] = paged.PagedBatch(
                _ptr(d["start"]), _ptr(d["seq_len"]), _ptr(d["table"]), len(d["n"]), d["T"],
                d["table"].shape[1], max(d["n"]), max(d["lens"]))
            need = paged.attention_scored_workspace_bytes(d["cache"], d["batch"], d["scores"], H)
    d["ws"] = torch.empty(max(need, 16), device=DEV, dtype=torch.uint8)


# ------------------------------------------------------------------ one pass

def _run_own(d):
    case, ws = d["case"], dict(workspace=d["ws"].data_ptr(), workspace_bytes=d["ws"].numel())
    if case["kind"] == "sample":
        _module("sampling").sample(
            case["act"], d["x"].data_ptr(), case["rows"], case["vocab"], d["u"].data_ptr(),
            d["tokens"].data_ptr(), how=d["how"], prob=d["prob"].data_ptr(), **ws)
        return d["tokens"], d["prob"]
    paged = _module("paged")
    if case["kind"] == "step":
        start, positions, seq, slots = d["out"]
        paged.plan(d["pool"], d["new"].data_ptr(), d["T"], case["context"], start.data_ptr(),
                   positions=positions.data_ptr(), token_seq=seq.data_ptr(),
                   slots=slots.data_ptr(), **ws)
        paged.release(d["pool"], d["keep"].data_ptr(), **ws)
        return (*d["out"], d["len"], d["table"], d["free"], d["n_free"])
    H, KV, hd = SHAPES[case["shape"]]
    q, k, v = d["q"], d["k"], d["v"]
    if case["kind"] == "paged":
        paged.attention_scored(d["cache"], d["batch"], d["scores"], q.data_ptr(),
                               d["out"].data_ptr(), H, case["act"], q_row_stride=q.stride(0), **ws)
    else:
        paged.attention_packed_scored(
            case["act"], d["scores"], q.data_ptr(), k.data_ptr(), v.data_ptr(),
            d["start"].data_ptr(), len(d["n"]), d["T"], max(d["n"]), H, KV, hd,
            d["out"].data_ptr(), q_row_stride=q.stride(0), k_row_stride=k.stride(0),
            v_row_stride=v.stride(0), **ws)
    return d["out"]


def _plain_plan(d):
    """New pages and token rows of the sequences that fit."""
    P, table, free, length = d["case"]["page"], d["table"], d["free"], d["len"].long()
    new = d["new"].long()
    held = (length + P - 1) // P
    need = (length + new + P - 1) // P - held
    pages, rows, left = torch.cumsum(need, 0), torch.cumsum(new, 0), d["n_free"].long()
    ok = ((need == 0) | (pages <= left)) & (rows <= d["T"])
    base = pages - need
    new, need = new * ok, need * ok
    start = torch.cumsum(torch.cat([new.new_zeros(1), new]), 0)
    t = torch.arange(d["T"], device=DEV)
    there = t < start[-1]
    s = (torch.searchsorted(start, t, right=True) - 1).clamp_max(len(new) - 1)
    pos = length[s] + t - start[s]
    j = pos // P
    fresh = there & (j >= held[s])
    popped = free[(left - 1 - base[s] - (j - held[s])).clamp(0, len(free) - 1)]
    at = s * table.shape[1] + j.clamp_max(table.shape[1] - 1)
    page = torch.where(fresh, popped, table.view(-1)[at])
    whole = torch.cat([table.view(-1), table.new_zeros(1)])
    whole[torch.where(fresh & (pos % P == 0), at, len(whole) - 1)] = page
    table.copy_(whole[:-1].view_as(table))
    d["out"][0].copy_(start)
    for out, x in zip(d["out"][1:], (pos, s, page.long() * P + pos % P)):
        out.copy_(torch.where(there, x.to(out.dtype), out))
    d["len"].copy_(length + new)
    d["n_free"].copy_(left - need.sum())


def _plain_release(d):
    """Pages past those that `keep` positions need, back to the free ones."""
    P, table, keep = d["case"]["page"], d["table"], d["keep"].long()
    kept, held = (keep + P - 1) // P, (d["len"].long() + P - 1) // P
    gone = held - kept
    total = d["n_free"].long() + gone.sum()
    col = torch.arange(table.shape[1], device=DEV)
    out = (col >= kept[:, None]) & (col < held[:, None])
    at = total - 1 - ((torch.cumsum(gone, 0) - gone)[:, None] + col - kept[:, None])
    free = torch.cat([d["free"], d["free"].new_zeros(1)])
    free[torch.where(out, at, len(free) - 1)] = table
    d["free"].copy_(free[:-1])
    table.masked_fill_(out, -1)
    d["len"].copy_(keep)
    d["n_free"].copy_(total)


def _plain_sample(d):
    x = d["x"].float()
    xs, idx = torch.sort(x, dim=-1, descending=True, stable=True)
    t, k, p, m, u = (d[n].double()[:, None] for n in ("t", "k", "p", "m", "u"))
    w = xs.double().sub_(xs[:, :1].double()).div_(torch.where(t > 0, t, 1.0)).exp_()
    c = torch.cumsum(w, -1)
    V = x.shape[1]
    nk = torch.where(k > 0, k, V).clamp_max(V).long()
    ck = c.gather(1, nk - 1)
    n_p = torch.where(p < 1, (c < p * ck).sum(-1, keepdim=True) + 1, nk)
    n_m = (w >= m).sum(-1, keepdim=True)
    n = torch.minimum(torch.minimum(nk, n_p), n_m).clamp_min(1)
    n = torch.where(t > 0, n, 1)
    cn = c.gather(1, n - 1)
    j = torch.minimum((c <= u * cn).sum(-1, keepdim=True), n - 1)
    d["tokens"].copy_(idx.gather(1, j)[:, 0])
    d["prob"].copy_((w.gather(1, j) / cn)[:, 0])
    return d["tokens"], d["prob"]


def _attend(q, k, v, pos, lo, hi, scale, cap, slopes):
    """q [S, N, H, hd] at positions pos [S, N], each over positions lo .. hi of k and v
    [S, L, KV, hd], all fp32."""
    S, N, H, hd = q.shape
    L, KV = k.shape[1], k.shape[2]
    G = H // KV
    q = q.view(S, N, KV, G, hd).permute(0, 2, 3, 1, 4).reshape(S, KV, G * N, hd)
    k = k.permute(0, 2, 3, 1).contiguous()
    w = torch.matmul(q, k).view(S, KV, G, N, L)
    w.mul_(scale)
    if cap:
        w.div_(cap).tanh_().mul_(cap)
    j = torch.arange(L, device=DEV)
    if slopes is not None:
        w.sub_((pos[..., None] - j).abs().float()[:, None, None] *
               slopes.view(KV, G)[None, :, :, None, None])
    unseen = (j < lo[..., None]) | (j > hi[..., None])
    w.masked_fill_(unseen[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = w.sum(-1, keepdim=True)
    w.div_(torch.where(total == 0, 1.0, total))
    o = torch.matmul(w.view(S, KV, G * N, L), v.permute(0, 2, 1, 3).contiguous())
    return o.view(S, KV, G, N, hd).permute(0, 3, 1, 2, 4).reshape(S, N, H, hd)


def _plain_attention(d):
    case = d["case"]
    H, KV, hd = SHAPES[case["shape"]]
    T, start = d["T"], d["start"].long()
    q = d["q"].float().view(T, H, hd)
    t = torch.arange(T, device=DEV)
    s = torch.searchsorted(start, t, right=True) - 1
    count = start[1:] - start[:-1]
    # sequences side by side, each padded to the longest
    n = torch.arange(max(d["n"]), device=DEV)
    at = (start[:-1, None] + n).clamp_max(T - 1)
    if case["kind"] == "paged":
        length = d["seq_len"].long()
        L = d["table"].shape[1] * case["page"]
        ks = d["kp"][d["table"].long()].view(-1, L, KV, hd).float()
        vs = d["vp"][d["table"].long()].view(-1, L, KV, hd).float()
    else:
        length = count
        ks, vs = (d[x].float().view(T, KV, hd)[at] for x in ("k", "v"))
    pos = (length - count)[:, None] + n
    lo = torch.zeros_like(pos) if d["first"] is None else d["first"].long()[at]
    hi = pos
    if case["window"]:
        lo = torch.maximum(lo, pos - case["window"] + 1)
    if d["prefix"] is not None:
        hi = torch.maximum(pos, torch.minimum(d["prefix"].long(), length)[:, None] - 1)
    o = _attend(q[at], ks, vs, pos, lo, hi, 1.0 / math.sqrt(hd), case["cap"], d["slopes"])
    d["out"].copy_(o[s, t - start[s]])
    return d["out"]


def _run_plain(d):
    if d["case"]["kind"] == "sample":
        return _plain_sample(d)
    if d["case"]["kind"] == "step":
        _plain_plan(d)
        _plain_release(d)
        return (*d["out"], d["len"], d["table"], d["free"], d["n_free"])
    return _plain_attention(d)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ what it cannot do without

def work(case):
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * SIZE[case["act"]] + 28),
                "flops": 2 * case["rows"] * case["vocab"]}
    n, lens = _lengths(case)
    T = sum(n)
    if case["kind"] == "step":
        P = case["page"]
        pages = sum(-(-m // P) - -(-(m - k) // P) for k, m in zip(n, lens))
        # lengths, counts, starts, what is kept; rows; page ids popped, entered, given back
        return {"bytes": 28 * len(n) + 16 * T + 20 * pages, "flops": 4 * T}
    H, KV, hd = SHAPES[case["shape"]]
    a, c = SIZE[case["act"]], SIZE[case["cache"]]
    prefix, first = _masks(case, n, lens)
    rows = pairs = t = 0
    for s, (k, m) in enumerate(zip(n, lens)):
        low, high = m, 0
        for p in range(m - k, m):
            lo = max(0 if first is None else first[t], p - case["window"] + 1 if case["window"]
                     else 0)
            hi = max(p, prefix[s] - 1) if prefix else p
            pairs += hi - lo + 1
            low, high = min(low, lo), max(high, hi + 1)
            t += 1
        rows += high - low
    table = 0 if case["kind"] == "packed" else 4 * (rows // case["page"] + len(n))
    return {"bytes": 2 * a * T * H * hd + 2 * c * rows * KV * hd + table + 8 * len(n),
            "flops": 4 * hd * H * pairs}


# ------------------------------------------------------------------ 64 bits, one row or head at a time

def _exact_sample(case, seed):
    d = _sample_inputs(case, seed)
    tokens, probs = [], []
    for r in range(case["rows"]):
        x = d["x"][r].double()
        t, k, p, m, u = (float(d[n][r]) for n in ("t", "k", "p", "m", "u"))
        if t == 0:
            tokens.append(x.argmax())
            probs.append(x.new_ones(()))
            continue
        order = torch.argsort(-x, stable=True)
        q = torch.softmax(x / t, -1)[order]
        if k > 0:
            q = q[:int(k)]
        keep = q >= m * q[0]
        if p < 1:  # what lies before a token has not yet reached p of the whole
            before = torch.cumsum(q, 0) - q
            keep &= before < p * q.sum()
        keep[0] = True
        q = q * keep
        j = int((torch.cumsum(q, 0) <= u * q.sum()).sum())
        tokens.append(order[min(j, int(keep.sum()) - 1)])
        probs.append(q[min(j, int(keep.sum()) - 1)] / q.sum())
    return torch.stack(tokens).to(torch.int32), torch.stack(probs)


def exact(case, seed):
    if case["kind"] == "step":
        return None  # whole numbers
    if case["kind"] == "sample":
        return _exact_sample(case, seed)
    d = _attention_inputs(case, seed)
    H, KV, hd = SHAPES[case["shape"]]
    q, out = d["q"].double().view(-1, H, hd), []
    k, v = d["k"].double().view(-1, KV, hd), d["v"].double().view(-1, KV, hd)
    for s, (n, m) in enumerate(zip(d["n"], d["lens"])):
        t0 = sum(d["n"][:s])
        qs, ks, vs = q[t0:t0 + n], k[t0:t0 + n], v[t0:t0 + n]
        if case["kind"] == "paged":
            pages = d["table"][s].long()[:-(-m // case["page"])]
            ks, vs = (x[pages].double().reshape(-1, KV, hd)[:m] for x in (d["kp"], d["vp"]))
        away = torch.arange(m - n, m, device=DEV)[:, None] - torch.arange(m, device=DEV)
        seen = away >= 0
        if d["prefix"] is not None:
            inside = torch.arange(m, device=DEV) < d["prefix"][s]
            seen |= inside[m - n:, None] & inside[None]
        if case["window"]:
            seen &= away < case["window"]
        if d["first"] is not None:
            seen &= torch.arange(m, device=DEV) >= d["first"][t0:t0 + n, None]
        o = torch.empty_like(qs)
        for h in range(H):
            sc = qs[:, h] @ ks[:, h // (H // KV)].T.contiguous() / math.sqrt(hd)
            if case["cap"]:
                sc = case["cap"] * torch.tanh(sc / case["cap"])
            if d["slopes"] is not None:
                sc = sc - float(d["slopes"][h]) * away.abs()
            w = torch.softmax(sc.where(seen, sc.new_tensor(-math.inf)), -1)
            o[:, h] = torch.nan_to_num(w) @ vs[:, h // (H // KV)].contiguous()
        out.append(o)
    return torch.cat(out)
