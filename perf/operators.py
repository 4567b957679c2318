"""Workloads of the paged cache and its attention, as measured cases.

Three operators of libkv-compact.so (include/kvc-cache.h):

  prompt   causal attention over packed prompts with grouped heads
  cells    attention of new tokens, or of a tree of drafted ones, over a paged
           cache with the per-head bias that a compaction fits
  pages    the cache's own steps: sharing a prompt between samples, drafting
           and accepting, compacting a sequence to the kept cells

Each is computed in plain torch operations, or by the library where `own` is
set. Shapes are those of this repository's benchmark and tests: 8 KV heads x
128 with 32 layers, 256-wide and 64-wide heads, 100k-token caches at 20% kept,
Q8_0 rows. Keys are N(0, 1) times a per-channel LogNormal(0, 0.5) scale, values
N(0, 1), queries a key of their sequence plus noise, so that rows attend some
cells far more than others.
"""
from __future__ import annotations

import ctypes
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

F32, F16, Q8_0, BF16 = 0, 1, 8, 30
CODE = {"f32": F32, "f16": F16, "q8_0": Q8_0, "bf16": BF16}
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NEG = float("-inf")


# ------------------------------------------------------------------- cases

def listed():
    return [
        # four short questions packed into one batch: the smallest, where launches count
        dict(name="prompt_short", entry="prompt", type="bf16", n_seq=4, n_tok=203, H=8, G=4, d=128, mix=1),
        # an ordinary prefill batch: ragged prompts of a 32-head model
        dict(name="prompt_packed", entry="prompt", type="bf16", n_seq=12, n_tok=16384, H=8, G=4, d=128, mix=2),
        # one long prompt, before its cache is compacted
        dict(name="prompt_long", entry="prompt", type="bf16", n_seq=1, n_tok=16384, H=8, G=4, d=128, mix=3),
        # 256-wide heads of a hybrid-attention model, odd lengths, F16
        dict(name="prompt_wide", entry="prompt", type="f16", n_seq=3, n_tok=5003, H=4, G=2, d=256, mix=4),
        # the next token of one chat: latency
        dict(name="decode_one", entry="cells", type="bf16", cache="bf16", n_seq=1, new=1, cells=4096, H=8, G=4, d=128,
             page=64, mix=5),
        # the next token of a full serving batch with ragged contexts
        dict(name="decode_batch", entry="cells", type="bf16", cache="bf16", n_seq=64, new=1, cells=16384, H=8, G=4,
             d=128, page=64, mix=6),
        # one 100k-token F32 cache compacted to 20%, with its fitted bias
        dict(name="decode_f32_bias", entry="cells", type="f32", cache="f32", n_seq=1, new=1, cells=20000, H=8, G=1,
             d=128, page=64, bias=1, mix=7),
        # drafts of 32 tokens verified over compacted F16 caches with bias
        dict(name="tree_bias", entry="cells", type="f16", cache="f16", n_seq=8, new=32, cells=20000, H=8, G=4, d=128,
             page=32, bias=1, tree=1, mix=8),
        # drafts of 13 tokens over long Q8_0 caches
        dict(name="tree_q8", entry="cells", type="bf16", cache="q8_0", n_seq=16, new=13, cells=32768, H=8, G=4, d=128,
             page=64, tree=1, mix=9),
        # 64 samples of 8 prompts start: prompts shared, their last pages copied, one token each
        dict(name="samples_start", entry="samples", type="bf16", L=32, n_seq=8, fan=8, new=1, cells=1000, H=8, d=128,
             page=64, mix=10),
        # drafts dropped, new ones written and some of them accepted, all layers
        dict(name="accept_drafts", entry="accept", type="f16", L=32, n_seq=16, new=13, cells=500, H=8, d=128, page=64,
             bias=1, mix=11),
        # a shared 32k-token prompt compacted to 20% for one of its users: refitted values, bias
        dict(name="compact_32k", entry="compact", type="bf16", L=32, n_seq=1, cells=32768, H=8, d=128, page=64, bias=1,
             ratio=0.2, mix=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    entry = rng.choice(["prompt", "prompt", "cells", "cells", "cells", "samples", "accept", "compact"])
    while True:
        c = dict(entry=entry, H=rng.choice([1, 2, 4, 8]), d=rng.choice([32, 64, 96, 128, 128, 256]),
                 mix=rng.randrange(1 << 30))
        if entry == "prompt":
            c.update(type=rng.choice(["bf16", "bf16", "f16", "f16", "f32"]), n_seq=_log(rng, 1, 32),
                     n_tok=_log(rng, 48, 16384), G=rng.choice([1, 2, 4, 8]))
            lens = _lens(c)
            if max(lens) ** 2 * c["n_seq"] * c["H"] * c["G"] * c["d"] > 16384.0 ** 2 * 32 * 128 / 2:
                continue
            if c["type"] == "f32" and sum(n * n for n in lens) * c["H"] * c["G"] * c["d"] > 4096.0 ** 2 * 32 * 128:
                continue
            return c
        c.update(page=rng.choice([16, 32, 64, 128, 256]), n_seq=_log(rng, 1, 64))
        if entry == "cells":
            cache = rng.choice(["bf16", "f16", "q8_0", "f32"])
            c.update(cache=cache, type=rng.choice(["bf16", "f16"]) if cache == "q8_0" else cache,
                     new=rng.choice([1, 1, _log(rng, 2, 64)]), cells=_log(rng, 32, 100000), G=rng.choice([1, 2, 4, 8]))
            if rng.random() < 0.5:
                c["bias"] = 1
            if c["new"] > 1 and rng.random() < 0.7:
                c["tree"] = 1
            if c["n_seq"] * c["cells"] * c["H"] * c["d"] > 64 * 16384 * 1024 // 2 or c["cells"] < c["new"]:
                continue
            if c["n_seq"] * c["cells"] * c["new"] * c["H"] * c["G"] > 8 * 20000 * 32 * 32:
                continue
            return c
        c.update(type=rng.choice(["bf16", "f16", "f32"]), L=_log(rng, 1, 32))
        if rng.random() < 0.5:
            c["bias"] = 1
        if entry == "samples":
            c.update(n_seq=_log(rng, 1, 16), fan=rng.choice([1, 2, 4, 8]), new=_log(rng, 1, 40),
                     cells=_log(rng, 8, 1000))
        elif entry == "accept":
            c.update(n_seq=_log(rng, 1, 32), new=_log(rng, 2, 64), cells=_log(rng, 8, 1000))
        else:
            c.update(n_seq=1, cells=_log(rng, 64, 32768), ratio=rng.choice([0.1, 0.2, 0.3, 0.5, 0.8]))
        rows = c["n_seq"] * (c["cells"] + c["page"] + c.get("fan", 1) * (c.get("new", 0) + 2 * c["page"]))
        if rows * c["L"] * c["H"] * c["d"] * (2 if c["type"] == "f32" else 1) > 32768 * 32 * 1024 // 2:
            continue
        return c


def _lens(c):
    """Ragged lengths of the sequences: a prompt batch sums to n_tok, a cache batch has at most `cells` each."""
    r = random.Random(c["mix"])
    n = c["n_seq"]
    if c["entry"] != "prompt":
        return [c["cells"] if i == 0 else max(c.get("new", 1), int(c["cells"] * r.uniform(0.2, 1.0))) for i in range(n)]
    w = [math.exp(r.gauss(0, 0.5)) for _ in range(n)]
    lens = [int(c["n_tok"] * x / sum(w)) for x in w]
    if n > 4:
        lens[1], lens[2] = 0, 1   # an empty request, and one of a single token
    lens[0] += c["n_tok"] - sum(lens)
    return lens


def _news(c):
    """New tokens of each sequence: `new` in the first, fewer in some of the others."""
    r = random.Random(c["mix"] + 1)
    return [c["new"] if i == 0 or r.random() < 0.5 else r.randint(1, c["new"]) for i in range(c["n_seq"])]


def _tree_masks(c, news):
    """Bit j of row i: drafted token i sees drafted token j (its ancestors and itself)."""
    r = random.Random(c["mix"] + 2)
    rows = []
    for n in news:
        seen = []
        for i in range(n):
            parent = r.randrange(max(0, i - 4), i) if i and r.random() < 0.9 else -1
            seen.append((1 << i) | (seen[parent] if parent >= 0 else 0))
        rows += seen
    return [b - (1 << 64) if b >> 63 else b for b in rows]


# ------------------------------------------------------------------ inputs

def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cu(lens):
    return _ints([0] + list(np.cumsum(lens)))


def _rows(gen, *shape):
    """N(0, 1) keys with a scale per channel (all but the first axes)."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    return x.mul_(torch.exp(0.5 * torch.randn(*shape[-2:], generator=gen, device="cuda")))


def _q8(x):
    """fp32 [..., n] -> Q8_0 bytes [..., n / 32 * 34]."""
    b = x.unflatten(-1, (-1, 32))
    d = b.abs().amax(-1, keepdim=True) / 127.0
    q = torch.round(b / d.clamp_min(1e-30)).clamp_(-127.0, 127.0).to(torch.int8).view(torch.uint8)
    return torch.cat([d.half().view(torch.uint8), q], -1).flatten(-2)


def _q8_values(b, double=False):
    b = b.unflatten(-1, (-1, 34))
    d, q = b[..., :2].contiguous().view(torch.float16), b[..., 2:].contiguous().view(torch.int8)
    return ((d.double() * q.double()) if double else (d.float() * q.float())).flatten(-2)


def _pool(gen, kind, L, pages, page, H, d, keys):
    x = torch.empty(L, pages, page, H, d, dtype=TORCH.get(kind, torch.float32), device="cuda")
    for l in range(L):
        x[l] = _rows(gen, pages, page, H, d) if keys else torch.randn(pages, page, H, d, generator=gen, device="cuda")
    return _q8(x.flatten(-2)) if kind == "q8_0" else x.flatten(-2)


def _table(gen, lens, page, n_pages, max_seqs, max_pages):
    """Pages of the first sequences, in a shuffled order, and the reference counts."""
    order = torch.randperm(n_pages, generator=gen, device="cuda").cpu().numpy()
    table = np.full((max_seqs, max_pages), -1, np.int32)
    refs = np.zeros(n_pages, np.int32)
    at = 0
    for s, n in enumerate(lens):
        k = -(-n // page)
        table[s, :k] = order[at:at + k]
        at += k
    refs[order[:at]] = 1
    full = np.zeros(max_seqs, np.int32)
    full[:len(lens)] = lens
    return _ints(table), _ints(full), _ints(refs)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=c)
    lens = _lens(c)
    H, d = c["H"], c["d"]
    if c["entry"] == "prompt":
        n, Hq, t = c["n_tok"], H * c["G"], TORCH[c["type"]]
        k = _rows(gen, n, H, d)
        near = (torch.rand(n, generator=gen, device="cuda") * torch.arange(n, device="cuda")).long()
        q = 0.5 * k[near].repeat_interleave(c["G"], 1) + torch.randn(n, Hq, d, generator=gen, device="cuda")
        v = torch.randn(n, H, d, generator=gen, device="cuda")
        s.update(q=q.to(t), k=k.to(t), v=v.to(t), cu=_cu(lens), o=torch.zeros(n, Hq, d, dtype=t, device="cuda"),
                 lse=torch.zeros(n, Hq, device="cuda"))
        torch.cuda.synchronize()
        return s
    page = c["page"]
    if c["entry"] == "cells":
        news = _news(c)
        need = sum(-(-n // page) for n in lens)
        max_pages = -(-max(lens) // page)
        n_pages = need + 3
        table, full, refs = _table(gen, lens, page, n_pages, c["n_seq"], max_pages)
        n, t, Hq = sum(news), TORCH[c["type"]], H * c["G"]
        K = _pool(gen, c["cache"], 1, n_pages, page, H, d, True)
        seen = (K if c["cache"] != "q8_0" else _q8_values(K)).reshape(-1, H, d)
        near = torch.randint(0, seen.shape[0], (n,), generator=gen, device="cuda")
        q = 0.5 * seen[near].float().repeat_interleave(c["G"], 1) + torch.randn(n, Hq, d, generator=gen, device="cuda")
        s.update(L=1, table=table, len=full, refs=refs, K=K, V=_pool(gen, c["cache"], 1, n_pages, page, H, d, False),
                 q=q.to(t), cu=_cu(news), seqs=_ints(list(range(c["n_seq"]))),
                 o=torch.zeros(n, Hq, d, dtype=t, device="cuda"), lse=torch.zeros(n, Hq, device="cuda"), bias=None,
                 mask=None, lens=lens, news=news)
        if c.get("bias"):
            # beta = log of the fitted masses, a few of them at the fit's floor of 1e-12
            s["bias"] = torch.randn(1, n_pages, H, page, generator=gen, device="cuda")
            s["bias"].masked_fill_(torch.rand(s["bias"].shape, generator=gen, device="cuda") < 0.05, math.log(1e-12))
        if c.get("tree"):
            s["mask"] = torch.tensor(_tree_masks(c, news), dtype=torch.int64, device="cuda")
        torch.cuda.synchronize()
        return s
    # pages
    L, t = c["L"], c["type"]
    n, fan = c["n_seq"], c.get("fan", 1)
    news = _news(c) if "new" in c else [0] * n
    grow = [-(-(m + c.get("new", 0)) // page) + 1 for m in lens]
    need = sum(grow) + n * fan * (2 + -(-c.get("new", 0) // page))
    if c["entry"] == "compact":
        need += grow[0]
    children = [n + i for i in range(n * fan)]
    table, full, refs = _table(gen, lens, page, need, n + n * fan, max(grow) + 1)
    s.update(L=L, table=table, len=full, refs=refs, K=_pool(gen, t, L, need, page, H, d, True),
             V=_pool(gen, t, L, need, page, H, d, False), bias=None, lens=lens, news=news)
    if c.get("bias"):
        s["bias"] = torch.randn(L, need, H, page, generator=gen, device="cuda")
    if c["entry"] == "samples":
        counts = [news[i % n] for i in range(n * fan)]
        m = sum(counts)
        s.update(src=_ints([i % n for i in range(n * fan)]), dst=_ints(children), count=_ints(counts), cu=_cu(counts),
                 m=m, counts=counts)
    elif c["entry"] == "accept":
        m = sum(news)
        r = random.Random(c["mix"] + 3)
        kept = [sorted(r.sample(range(k), r.randint(0, min(k, 5)))) for k in news]
        flat = [x for k in kept for x in k]
        s.update(seqs=_ints(list(range(n))), count=_ints(news), cu=_cu(news), m=m, start=_ints(lens),
                 none=_cu([0] * n), idx=_ints(flat or [0]), kept=_cu([len(k) for k in kept]), n_idx=len(flat))
    else:
        m, T = 0, lens[0]
        k = max(1, int(np.float32(T) * np.float32(c["ratio"])))
        idx = torch.rand(L, T, generator=gen, device="cuda").topk(k, 1).indices.sort(1).values.int()
        s.update(src=_ints([0]), dst=_ints([1]), start=_ints([0]), kept=_cu([k]), idx=idx, n_idx=k,
                 values=torch.randn(L, k, H * d, generator=gen, device="cuda").to(TORCH[t]),
                 beta=torch.randn(L, H, k, generator=gen, device="cuda") if c.get("bias") else None)
    if m:
        s["k_new"] = _rows(gen, L, m, H, d).flatten(-2).to(TORCH[t])
        s["v_new"] = torch.randn(L, m, H * d, generator=gen, device="cuda").to(TORCH[t])
    s["status"] = torch.zeros(n * fan, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------- the plain operators

def _pad(cu, most):
    """Index [n][most] of each sequence's tokens, and which of them are there."""
    t = torch.arange(most, device="cuda")
    lens = (cu[1:] - cu[:-1]).long()
    there = t < lens[:, None]
    return torch.where(there, cu[:-1, None].long() + t, 0), there


def _attend(q, k, v, seen, bias, scale):
    """q [n][N][Hq][d], k and v [n][M][H][d], seen [n][N][M], bias [n][H][M] -> fp32 o [n][N][Hq][d], lse [n][N][Hq]."""
    n, N, Hq, d = q.shape
    M, H = k.shape[1], k.shape[2]
    G = Hq // H
    q = q.float().view(n, N, H, G, d).permute(0, 2, 3, 1, 4).reshape(n * H, G * N, d)
    k = k.float().permute(0, 2, 3, 1).reshape(n * H, d, M).contiguous()
    v = v.float().permute(0, 2, 1, 3).reshape(n * H, M, d).contiguous()
    S = torch.bmm(q, k).mul_(scale).view(n, H, G, N, M)
    if bias is not None:
        S += bias[:, :, None, None, :]
    S.masked_fill_(~seen[:, None, None], NEG)
    m = S.amax(-1, keepdim=True)
    S = S.sub_(m.masked_fill(m == NEG, 0.0)).exp_()
    l = S.sum(-1, keepdim=True)
    o = torch.bmm(S.view(n * H, G * N, M), v).view(n, H, G, N, d)
    o = o / torch.where(l > 0, l, 1.0)
    lse = (m + l.log()).view(n, H, G, N)
    return o.permute(0, 3, 1, 2, 4).reshape(n, N, Hq, d), lse.permute(0, 3, 1, 2).reshape(n, N, Hq)


def _plain_prompt(s):
    c = s["case"]
    most = max(_lens(c))
    at, there = _pad(s["cu"], most)
    t = torch.arange(most, device="cuda")
    seen = (t[None, :] <= t[:, None])[None] & there[:, None, :]
    o, lse = _attend(s["q"][at], s["k"][at], s["v"][at], seen, None, 1.0 / math.sqrt(c["d"]))
    s["o"].copy_(o[there])
    s["lse"].copy_(lse[there])
    return dict(o=s["o"], lse=s["lse"])


def _plain_cells(s):
    c = s["case"]
    page, H, d = c["page"], c["H"], c["d"]
    seqs = s["seqs"].long()
    most, new = max(s["lens"]), max(s["news"])
    at, there = _pad(s["cu"], new)
    pos = torch.arange(most, device="cuda")
    lens = s["len"][seqs].long()
    pages = s["table"][seqs].long()[:, pos // page].clamp_min(0)
    cell = pages * page + pos % page

    def rows(pool):
        x = pool[0].reshape(-1, pool.shape[-1])[cell]
        return (_q8_values(x) if c["cache"] == "q8_0" else x.float()).view(len(seqs), most, H, d)

    bias = None
    if s["bias"] is not None:
        bias = s["bias"][0].permute(0, 2, 1).reshape(-1, H)[cell].permute(0, 2, 1)
    rel = pos[None] - (lens - (s["cu"][1:] - s["cu"][:-1]).long())[:, None]   # [n][M], < 0: committed
    if s["mask"] is not None:
        bit = (s["mask"][at][:, :, None] >> rel.clamp(0, 63)[:, None, :]) & 1
        drafted = (bit == 1) & (rel < 64)[:, None, :]
    else:
        drafted = rel[:, None, :] <= torch.arange(new, device="cuda")[None, :, None]
    seen = ((rel < 0)[:, None, :] | drafted) & (pos[None] < lens[:, None])[:, None, :]
    o, lse = _attend(s["q"][at], rows(s["K"]), rows(s["V"]), seen, bias, 1.0 / math.sqrt(d))
    s["o"].copy_(o[there])
    s["lse"].copy_(lse[there])
    return dict(o=s["o"], lse=s["lse"])


def _drop(s, seqs, first):
    """The pages of seqs at table columns >= first [n] are given back."""
    t = s["table"][seqs]
    col = torch.arange(t.shape[1], device="cuda")
    gone = (col >= first[:, None]) & (t >= 0)
    s["refs"].index_add_(0, t[gone].long(), torch.full_like(t[gone], -1))
    s["table"][seqs] = torch.where(gone, -1, t)


def _take(s, seqs, first, need):
    """Fresh pages, lowest first: table columns first .. first + need - 1 of each sequence."""
    free = torch.nonzero(s["refs"] == 0)[:, 0]
    col = torch.arange(s["table"].shape[1], device="cuda")
    j = col - first[:, None]
    new = (j >= 0) & (j < need[:, None])
    page = free[torch.where(new, (need.cumsum(0) - need)[:, None] + j, 0)].int()
    s["table"][seqs] = torch.where(new, page, s["table"][seqs])
    s["refs"][page[new].long()] = 1


def _move(s, seqs, old, to, frm, use):
    """Cells frm -> to of each sequence ([n][k] or [L][n][k]), read through the table `old`, where `use`."""
    page, L = s["case"]["page"], s["L"]
    where = lambda t, x: torch.gather(t[seqs].long().expand(*x.shape[:-1], -1), -1, x // page) * page + x % page  # noqa: E731
    frm, to, use = (x.expand(L, *x.shape[-2:]).contiguous() for x in (frm, to, use))
    a, b = where(old, torch.where(use, frm, 0)), where(s["table"], torch.where(use, to, 0))
    l = torch.arange(L, device="cuda")[:, None, None].expand_as(a)[use]
    a, b = a[use], b[use]
    pools = [s["K"].view(L, -1, s["K"].shape[-1])]
    if "values" not in s:
        pools.append(s["V"].view(L, -1, s["V"].shape[-1]))
    for x in pools:
        x[l, b] = x[l, a]
    if s["bias"] is not None and s.get("beta") is None:
        h = torch.arange(s["bias"].shape[2], device="cuda")
        s["bias"][l[:, None], (b // page)[:, None], h, (b % page)[:, None]] = s["bias"][
            l[:, None], (a // page)[:, None], h, (a % page)[:, None]]


def _plain_fork(s):
    src, dst = s["src"].long(), s["dst"].long()
    _drop(s, dst, torch.zeros_like(dst))
    t = s["table"][src]
    s["table"][dst], s["len"][dst] = t, s["len"][src]
    s["refs"].index_add_(0, t[t >= 0].long(), torch.ones_like(t[t >= 0]))


def _plain_extend(s, seqs):
    page, count = s["case"]["page"], s["count"].long()
    old = s["len"][seqs].long()
    have = -(-old // page)
    last = (old // page).clamp_max(s["table"].shape[1] - 1)
    at_last = torch.gather(s["table"][seqs].long(), 1, last[:, None])[:, 0].clamp_min(0)
    copied = (old % page > 0) & (count > 0) & (s["refs"][at_last] > 1)
    before = s["table"].clone()
    _take(s, seqs, have - copied.long(), -(-(old + count) // page) - have + copied.long())
    s["refs"].index_add_(0, at_last, -copied.int())
    cell = torch.arange(page, device="cuda")
    cells = (last * page)[:, None] + cell
    _move(s, seqs, before, cells, cells, copied[:, None] & (cell < (old % page)[:, None]))
    s["len"][seqs] = (old + count).int()
    s["status"].zero_()


def _plain_write(s, seqs):
    page, m, L = s["case"]["page"], s["m"], s["L"]
    r = torch.arange(m, device="cuda")
    q = torch.searchsorted(s["cu"][1:].long(), r, right=True)
    pos = s["len"][seqs][q].long() - s["cu"][1:][q].long() + r
    cell = s["table"][seqs[q], pos // page].long() * page + pos % page
    s["K"].view(L, -1, s["K"].shape[-1])[:, cell] = s["k_new"]
    s["V"].view(L, -1, s["V"].shape[-1])[:, cell] = s["v_new"]
    if s["bias"] is not None:
        s["bias"].permute(0, 1, 3, 2)[:, cell // page, cell % page] = 0.0


def _plain_compact(s, seqs, kept, idx):
    """idx [L or 1][n_idx]."""
    page = s["case"]["page"]
    start, count = s["start"].long(), (kept[1:] - kept[:-1]).long()
    new = start + count
    t = s["table"][seqs].long()
    col = torch.arange(t.shape[1], device="cuda")
    kept_pages = -(-new // page)
    written = (count > 0)[:, None] & (col >= (start // page)[:, None]) & (col < kept_pages[:, None])
    shared = written & (s["refs"][t.clamp_min(0)] > 1)
    before = s["table"].clone()
    free = torch.nonzero(s["refs"] == 0)[:, 0]
    nth = shared.view(-1).cumsum(0).view(shared.shape) - 1
    fresh = free[torch.where(shared, nth, 0)]
    gone = shared | ((col >= kept_pages[:, None]) & (t >= 0))
    s["refs"].index_add_(0, t[gone], torch.full_like(t[gone], -1, dtype=torch.int32))
    s["refs"][fresh[shared]] = 1
    s["table"][seqs] = torch.where(shared, fresh, torch.where(gone, -1, t)).int()
    if idx is not None:
        most = s["n_idx"]
        at, there = _pad(kept, most)
        to = start[:, None] + torch.arange(most, device="cuda")
        _move(s, seqs, before, to, start[:, None] + idx[:, at].long(), there)
        # cells before start on a page that was replaced
        lead = torch.gather(shared, 1, (start // page).clamp_max(t.shape[1] - 1)[:, None])
        cell = torch.arange(page, device="cuda")
        cells = (start // page * page)[:, None] + cell
        _move(s, seqs, before, cells, cells, lead & (cell < (start % page)[:, None]))
        q = s["table"][seqs].long()
        cell = (torch.gather(q, 1, to // page) * page + to % page)[there]
        if "values" in s:
            s["V"].view(s["L"], -1, s["V"].shape[-1])[:, cell] = s["values"]
        if s.get("beta") is not None:
            s["bias"].permute(0, 1, 3, 2)[:, cell // page, cell % page] = s["beta"].permute(0, 2, 1)
    s["len"][seqs] = new.int()
    s["status"].zero_()


def _pages_out(s):
    out = {k: s[k] for k in ("K", "V", "table", "len", "refs", "status")}
    if s["bias"] is not None:
        out["bias"] = s["bias"]
    return out


def _plain_samples(s):
    _plain_fork(s)
    _plain_extend(s, s["dst"].long())
    _plain_write(s, s["dst"].long())
    return _pages_out(s)


def _plain_accept(s):
    seqs = s["seqs"].long()
    _plain_compact(s, seqs, s["none"], None)
    _plain_extend(s, seqs)
    _plain_write(s, seqs)
    _plain_compact(s, seqs, s["kept"], s["idx"][None])
    return _pages_out(s)


def _plain_compacting(s):
    _plain_fork(s)
    _plain_compact(s, s["dst"].long(), s["kept"], s["idx"])
    return _pages_out(s)


# ------------------------------------------------------- the library's calls

_dll = None


def _library():
    """libkv-compact.so with the cache's entry points declared."""
    global _dll
    if _dll is None:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "kv-compact_amd"))
        import kvcompact as kc
        _dll = kc, kc.bind_cache(kc.load_product().dll)
    return _dll


def _calls(s):
    """The structs and workspace that a program keeps beside its buffers."""
    kc, dll = _library()
    c = s["case"]
    p = lambda x: x.data_ptr() if x is not None else None  # noqa: E731
    H, d = c["H"], c["d"]
    if c["entry"] == "prompt":
        Hq = H * c["G"]
        return kc.PromptArgs(q=kc.Heads(p(s["q"]), Hq * d, d), k=kc.Heads(p(s["k"]), H * d, d),
                             v=kc.Heads(p(s["v"]), H * d, d), o=kc.Heads(p(s["o"]), Hq * d, d), lse=p(s["lse"]),
                             cu=p(s["cu"]), type=CODE[c["type"]], n_seq=c["n_seq"], n_tok=c["n_tok"], n_head=Hq,
                             n_head_kv=H, d_k=d, d_v=d), None, None
    code = CODE[c.get("cache", c["type"])]
    cache = kc.KvCache(n_layers=s["L"], n_pages=s["refs"].numel(), page_size=c["page"], max_seqs=s["len"].numel(),
                       max_pages=s["table"].shape[1], n_head_kv=H, d_k=d, d_v=d, k_type=code, v_type=code,
                       K=p(s["K"]), V=p(s["V"]), bias=p(s["bias"]), table=p(s["table"]), len=p(s["len"]),
                       refs=p(s["refs"]))
    if c["entry"] == "cells":
        Hq = H * c["G"]
        a = kc.CacheAttnArgs(q=kc.Heads(p(s["q"]), Hq * d, d), o=kc.Heads(p(s["o"]), Hq * d, d), lse=p(s["lse"]),
                             seqs=p(s["seqs"]), cu=p(s["cu"]), mask=p(s["mask"]), mask_words=1, layer=0,
                             type=CODE[c["type"]], n_seq=c["n_seq"], n_tok=s["q"].shape[0], n_head=Hq,
                             max_new=max(s["news"]), max_len=max(s["lens"]))
        n = dll.kvc_attn_cache_workspace(ctypes.byref(cache), ctypes.byref(a))
        return cache, a, torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    n = dll.kvc_cache_workspace(ctypes.byref(cache), s["status"].numel())
    rows = None
    if "k_new" in s:
        b = s["k_new"].element_size()
        rows = [kc.Rows(p(s[x]), s["m"] * H * d * b, H * d * b) for x in ("k_new", "v_new")]
    elif "values" in s:
        b = s["values"].element_size()
        k = s["n_idx"]
        rows = [kc.Values(p(s["values"]), k * H * d * b, H * d * b, d * b),
                kc.Betas(p(s["beta"]), H * k, k) if s.get("beta") is not None else None]
    return cache, rows, torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")


def _ok(rc, what):
    if rc:
        raise RuntimeError("%s returned %d" % (what, rc))


def _own(s):
    kc, dll = _library()
    if "calls" not in s:
        s["calls"] = _calls(s)
    c, (cache, a, ws) = s["case"], s["calls"]
    st = torch.cuda.current_stream().cuda_stream
    if c["entry"] == "prompt":
        _ok(dll.kvc_attn_prompt(cache, st), "kvc_attn_prompt")
        return dict(o=s["o"], lse=s["lse"])
    if c["entry"] == "cells":
        _ok(dll.kvc_attn_cache(cache, a, ws.data_ptr(), ws.numel(), st), "kvc_attn_cache")
        return dict(o=s["o"], lse=s["lse"])
    w = ws.data_ptr(), ws.numel(), st
    status = s["status"].data_ptr()

    def ptr(k):
        return s[k].data_ptr()

    if c["entry"] == "accept":
        n = c["n_seq"]
        seqs = ptr("seqs")
        _ok(dll.kvc_cache_compact(cache, n, seqs, ptr("start"), ptr("none"), 0, None, 0, None, None, status, *w), "cut")
        grown = seqs
    else:
        n = s["dst"].numel()
        grown = ptr("dst")
        _ok(dll.kvc_cache_free(cache, n, grown, st), "kvc_cache_free")
        _ok(dll.kvc_cache_fork(cache, n, ptr("src"), grown, status, st), "kvc_cache_fork")
    if c["entry"] == "compact":
        _ok(dll.kvc_cache_compact(cache, n, grown, ptr("start"), ptr("kept"), s["n_idx"], ptr("idx"), s["n_idx"], a[0],
                                  a[1], status, *w), "kvc_cache_compact")
        return _pages_out(s)
    _ok(dll.kvc_cache_extend(cache, n, grown, ptr("count"), status, *w), "kvc_cache_extend")
    _ok(dll.kvc_cache_write(cache, 0, s["L"], n, grown, ptr("cu"), s["m"], CODE[c["type"]], a[0], a[1], st),
        "kvc_cache_write")
    if c["entry"] == "accept":
        _ok(dll.kvc_cache_compact(cache, n, grown, ptr("start"), ptr("kept"), s["n_idx"], ptr("idx"), 0, None, None,
                                  status, *w), "kvc_cache_compact")
    return _pages_out(s)


def run(state):
    if own:
        return _own(state)
    plain = dict(prompt=_plain_prompt, cells=_plain_cells, samples=_plain_samples, accept=_plain_accept,
                 compact=_plain_compacting)
    return plain[state["case"]["entry"]](state)


# -------------------------------------------------------------------- work

def work(case):
    c = case
    H, d, lens = c["H"], c["d"], _lens(c)
    size = {"f32": 4.0, "f16": 2.0, "bf16": 2.0, "q8_0": 34.0 / 32}
    if c["entry"] == "prompt":
        Hq, n = H * c["G"], c["n_tok"]
        return dict(bytes=size[c["type"]] * n * (2 * Hq + 2 * H) * d + 4.0 * n * Hq,
                    flops=sum(2.0 * d * Hq * m * (m + 1) for m in lens))
    news = _news(c) if "new" in c else None
    if c["entry"] == "cells":
        Hq = H * c["G"]
        cell = 2 * size[c["cache"]] * H * d + (4 * H if c.get("bias") else 0)
        q = sum(news)
        return dict(bytes=sum(lens) * cell + q * Hq * (2 * size[c["type"]] * d + 4) + 4.0 * sum(
            -(-m // c["page"]) for m in lens), flops=sum(4.0 * d * Hq * m * k for m, k in zip(lens, news)))
    cell = c["L"] * (2 * size[c["type"]] * H * d + (4 * H if c.get("bias") else 0))
    if c["entry"] == "samples":
        # the shared last pages' cells copied, the new rows read and written
        n = len(lens)
        moved = c["fan"] * sum((m % c["page"]) for m, k in zip(lens, news))
        return dict(bytes=2 * cell * (moved + c["fan"] * sum(news)), flops=0.0)
    if c["entry"] == "accept":
        return dict(bytes=2 * cell * (sum(news) + 2 * len(news)), flops=0.0)
    return dict(bytes=2 * cell * max(1, int(np.float32(lens[0]) * np.float32(c["ratio"]))), flops=0.0)


# ------------------------------------------------- 64-bit results for checking

def _exact_rows(q, k, v, seen, bias, scale):
    """One sequence: q [N][Hq][d], k and v [M][H][d] in 64 bits, seen [N][M]."""
    N, Hq, _ = q.shape
    H = k.shape[1]
    o = torch.zeros(N, Hq, v.shape[2], dtype=torch.float64, device="cuda")
    lse = torch.full((N, Hq), NEG, dtype=torch.float64, device="cuda")
    for h in range(Hq):
        g = h // (Hq // H)
        x = torch.matmul(q[:, h].contiguous(), k[:, g].t().contiguous()) * scale
        if bias is not None:
            x = x + bias[g]
        x = torch.where(seen, x, NEG)
        lse[:, h] = torch.logsumexp(x, 1)
        w = torch.exp(x - torch.where(lse[:, h] == NEG, 0.0, lse[:, h])[:, None])
        o[:, h] = torch.matmul(w, v[:, g].contiguous())
    return o, lse


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    scale = 1.0 / math.sqrt(c["d"])
    lens = _lens(c)
    if c["entry"] == "prompt":
        parts, at = [], 0
        for n in lens:
            i = torch.arange(n, device="cuda")
            q, k, v = (s[x][at:at + n].double() for x in "qkv")
            parts.append(_exact_rows(q, k, v, i[:, None] >= i, None, scale))
            at += n
        return dict(o=torch.cat([p[0] for p in parts]), lse=torch.cat([p[1] for p in parts]))
    page = c["page"]
    table = s["table"].cpu().numpy()
    if c["entry"] == "cells":
        bits = [int(b) & ((1 << 64) - 1) for b in s["mask"].cpu()] if s["mask"] is not None else None
        parts, at = [], 0
        for i, (n, new) in enumerate(zip(lens, s["news"])):
            pages = torch.tensor(table[i, :-(-n // page)], device="cuda").long()
            k, v = (s[x][0, pages].reshape(-1, s[x].shape[-1])[:n] for x in "KV")
            k, v = ((_q8_values(x, True) if c["cache"] == "q8_0" else x.double()).view(n, c["H"], c["d"]) for x in (k, v))
            b = s["bias"][0, pages].permute(1, 0, 2).reshape(c["H"], -1)[:, :n].double() if s["bias"] is not None else None
            see = [[(bits[at + a] >> j) & 1 if bits else j <= a for j in range(new)] for a in range(new)]
            seen = torch.ones(new, n, dtype=torch.bool, device="cuda")
            seen[:, n - new:] = torch.tensor(see, dtype=torch.bool, device="cuda").view(new, new)
            parts.append(_exact_rows(s["q"][at:at + new].double(), k, v, seen, b, scale))
            at += new
        return dict(o=torch.cat([p[0] for p in parts]), lse=torch.cat([p[1] for p in parts]))
    return _exact_pages(c, s, lens, table.tolist())


def _exact_pages(c, s, lens, table):
    """The pages' steps one after another on lists; cells copied in their own type."""
    page, L = c["page"], s["L"]
    table = [[p for p in row if p >= 0] for row in table]
    held = s["len"].cpu().tolist()
    refs = s["refs"].cpu().tolist()
    pools = {x: s[x].clone() for x in ("K", "V")}
    if s["bias"] is not None:
        pools["bias"] = s["bias"].permute(0, 1, 3, 2).contiguous()   # [L][page][cell][H]

    def spot(row, cells):
        return torch.tensor([row[x // page] * page + x % page for x in cells], device="cuda", dtype=torch.long)

    def flat(x):
        return x.reshape(L, -1, x.shape[-1])

    def copy(names, l, frm, to):
        for x in names:
            y = flat(pools[x])
            y[l, to] = y[l, frm].clone()

    def fork(src, dst):
        table[dst], held[dst] = list(table[src]), held[src]
        for p in table[src]:
            refs[p] += 1

    def extend(seqs, counts):
        was = list(refs)
        for q, k in zip(seqs, counts):
            old, row = held[q], table[q]
            free = [p for p, r in enumerate(was) if r == 0]
            if old % page and k and shared[row[-1]] > 1:
                p, cells = free.pop(0), range(old // page * page, old)
                frm = spot(row, cells)
                refs[row[-1]] -= 1
                row[-1] = p
                refs[p] = was[p] = 1
                for l in range(L):
                    copy(pools, l, frm, spot(row, cells))
            while len(row) * page < old + k:
                p = free.pop(0)
                row.append(p)
                refs[p] = was[p] = 1
            held[q] = old + k

    def write(seqs, counts):
        at = 0
        for q, k in zip(seqs, counts):
            to = spot(table[q], range(held[q] - k, held[q]))
            flat(pools["K"])[:, to] = s["k_new"][:, at:at + k]
            flat(pools["V"])[:, to] = s["v_new"][:, at:at + k]
            if "bias" in pools:
                flat(pools["bias"])[:, to] = 0.0
            at += k

    if c["entry"] in ("samples", "compact"):
        for a, b in zip(s["src"].cpu().tolist(), s["dst"].cpu().tolist()):
            fork(a, b)
    shared = list(refs)
    if c["entry"] == "samples":
        children = s["dst"].cpu().tolist()
        extend(children, s["counts"])
        write(children, s["counts"])
    elif c["entry"] == "accept":
        extend(range(c["n_seq"]), s["news"])
        write(range(c["n_seq"]), s["news"])
        cu, idx = s["kept"].cpu().tolist(), s["idx"].cpu().tolist()
        for q in range(c["n_seq"]):
            keep = idx[cu[q]:cu[q + 1]]
            to, frm = spot(table[q], [lens[q] + i for i in range(len(keep))]), spot(table[q], [lens[q] + x for x in keep])
            for l in range(L):
                copy(pools, l, frm, to)
            held[q] = lens[q] + len(keep)
            for p in table[q][-(-held[q] // page):]:
                refs[p] -= 1
            del table[q][-(-held[q] // page):]
    else:
        k = s["n_idx"]
        old = table[1]
        free = [p for p, r in enumerate(refs) if r == 0]
        for p in old:
            refs[p] -= 1
        table[1] = free[:-(-k // page)]
        for p in table[1]:
            refs[p] = 1
        held[1] = k
        to, idx = spot(table[1], range(k)), s["idx"].cpu().tolist()
        for l in range(L):
            frm = spot(old, idx[l])
            copy(["K"] + (["bias"] if "bias" in pools and s["beta"] is None else []), l, frm, to)
        flat(pools["V"])[:, to] = s["values"]
        if s["beta"] is not None:
            flat(pools["bias"])[:, to] = s["beta"].permute(0, 2, 1)
    width = s["table"].shape[1]
    out = dict(K=pools["K"].double(), V=pools["V"].double(), table=_ints([r + [-1] * (width - len(r)) for r in table]),
               len=_ints(held), refs=_ints(refs), status=torch.zeros_like(s["status"]))
    if "bias" in pools:
        out["bias"] = pools["bias"].permute(0, 1, 3, 2).double().contiguous()
    return out
