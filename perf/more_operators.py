"""Workloads of a cache that is kept to a budget, as measured cases.

Operators of libkv-compact.so (include/kvc-cache.h):

  prompt   causal attention over packed prompts in which a token sees the first
           tokens of its sequence and a sliding window of the last ones
  cells    the same for new or drafted tokens over a paged cache
  weigh    the softmax weight that tokens give each cell, added to what the
           cell has gathered
  evict    the cells that gathered the most picked for every layer, and their
           weights moved to a sequence that goes on with those cells

Each is computed in plain torch operations, or by the library where `own` is
set. Shapes are those of this repository's benchmark and tests: 8 KV heads x
128 with 32 layers, 256-wide heads, prompts of 16384 tokens, caches of 16384 to
32768 cells, 20% kept, Q8_0 rows. Keys are N(0, 1) times a per-channel
LogNormal(0, 0.5) scale, values N(0, 1), queries a key of their sequence plus
noise, so that rows attend some cells far more than others.
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
NO_WINDOW = 1 << 30


# ------------------------------------------------------------------- cases

def listed():
    return [
        # four short questions packed into one batch: the smallest, where launches count
        dict(name="window_prompt_short", entry="prompt", type="bf16", n_seq=4, n_tok=203, first=4, last=64, H=8, G=4,
             d=128, mix=1),
        # an ordinary prefill batch of a 32-head model with a window of 1024
        dict(name="window_prompt_packed", entry="prompt", type="bf16", n_seq=12, n_tok=16384, first=4, last=1024, H=8,
             G=4, d=128, mix=2),
        # one long document under a window of 4096
        dict(name="window_prompt_long", entry="prompt", type="bf16", n_seq=1, n_tok=32768, first=4, last=4096, H=8,
             G=4, d=128, mix=3),
        # 256-wide heads of a hybrid-attention model: its window layers have no first tokens; odd lengths, F16
        dict(name="window_prompt_wide", entry="prompt", type="f16", n_seq=3, n_tok=5003, first=0, last=512, H=4, G=2,
             d=256, mix=4),
        # the next token of one long chat: latency
        dict(name="window_decode_one", entry="cells", type="bf16", cache="bf16", n_seq=1, new=1, cells=20000, first=4,
             last=1024, H=8, G=4, d=128, page=64, mix=5),
        # the next token of a full serving batch with ragged contexts
        dict(name="window_decode_batch", entry="cells", type="bf16", cache="bf16", n_seq=64, new=1, cells=16384,
             first=16, last=4096, H=8, G=4, d=128, page=64, mix=6),
        # drafts of 13 tokens over long Q8_0 caches
        dict(name="window_tree_q8", entry="cells", type="bf16", cache="q8_0", n_seq=16, new=13, cells=32768, first=4,
             last=2048, H=8, G=4, d=128, page=64, tree=1, mix=7),
        # weights gathered beside each decoded token of a serving batch
        dict(name="weigh_decode", entry="weigh", type="bf16", cache="bf16", n_seq=64, new=1, cells=16384, decay=1.0,
             H=8, G=4, d=128, page=64, mix=8),
        # the last 32 tokens of eight prompts decide which cells matter; F16 caches with a fitted bias
        dict(name="weigh_last_tokens", entry="weigh", type="f16", cache="f16", n_seq=8, new=32, cells=20000, decay=0.0,
             H=8, G=4, d=128, page=32, bias=1, mix=9),
        # every token of a prompt counted, behind its attention
        dict(name="weigh_prompt", entry="weigh", type="bf16", cache="bf16", n_seq=1, new=16384, cells=16384, decay=0.0,
             H=8, G=4, d=128, page=64, mix=10),
        # a chat that reached its limit goes back to its budget of 4096 cells, all layers
        dict(name="evict_one", entry="evict", L=32, n_seq=1, cells=5120, first=4, keep=4092, recent=512, H=8, page=64,
             mix=11),
        # sixteen ragged contexts cut to a fifth of 32768 cells, all layers
        dict(name="evict_batch", entry="evict", L=32, n_seq=16, cells=32768, first=4, keep=6549, recent=256, H=8,
             page=64, mix=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    entry = rng.choice(["prompt", "prompt", "cells", "cells", "weigh", "weigh", "evict"])
    while True:
        c = dict(entry=entry, H=rng.choice([1, 2, 4, 8]), mix=rng.randrange(1 << 30))
        first = rng.choice([0, 1, 4, 16, _log(rng, 1, 200)])
        if entry == "evict":
            c.update(L=_log(rng, 1, 32), n_seq=_log(rng, 1, 16), cells=_log(rng, 16, 32768), first=first,
                     recent=_log(rng, 1, 512), page=rng.choice([16, 32, 64, 128, 256]))
            c["keep"] = max(1, int(c["cells"] * rng.choice([0.1, 0.2, 0.3, 0.5, 0.8])))
            if rng.random() < 0.3:
                c["most"] = 1
            if rng.random() < 0.3:
                c["shared"] = 1
            return c
        c.update(G=rng.choice([1, 2, 4, 8]), d=rng.choice([32, 64, 96, 128, 128, 256]))
        if entry == "prompt":
            c.update(type=rng.choice(["bf16", "bf16", "f16", "f16", "f32"]), n_seq=_log(rng, 1, 32),
                     n_tok=_log(rng, 48, 32768), first=first, last=_log(rng, 1, 4096))
            pairs = float(c["n_tok"]) * (c["last"] + c["first"] + 64) * c["H"] * c["G"] * c["d"]
            if pairs > 32768.0 * 4096 * 32 * 128 / (16 if c["type"] == "f32" else 1):
                continue
            return c
        cache = rng.choice(["bf16", "f16", "q8_0", "f32"])
        c.update(cache=cache, type=rng.choice(["bf16", "f16"]) if cache == "q8_0" else cache,
                 page=rng.choice([16, 32, 64, 128, 256]), n_seq=_log(rng, 1, 64), cells=_log(rng, 32, 100000),
                 new=rng.choice([1, 1, _log(rng, 2, 64)]))
        if c["n_seq"] * c["cells"] * c["H"] * c["d"] > 64 * 16384 * 1024 // 2 or c["cells"] < c["new"]:
            continue
        if rng.random() < 0.5:
            c["bias"] = 1
        if entry == "cells" or rng.random() < 0.3:
            c.update(first=first, last=_log(rng, 1, 8192))
        if entry == "weigh":
            c["decay"] = rng.choice([0.0, 1.0, 0.9375])
            if rng.random() < 0.2:
                c.update(n_seq=min(c["n_seq"], 4), cells=min(c["cells"], 4096))
                c["new"] = c["cells"]
            elif c["new"] > 2 and rng.random() < 0.3:
                c["tail"] = rng.randint(1, c["new"])
        if 1 < c["new"] <= 64 and rng.random() < 0.7:
            c["tree"] = 1
        if c["n_seq"] * c["cells"] * c["new"] * c["H"] * c["G"] > 8 * 20000 * 32 * 32:
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


def _keeps(c):
    """Cells each sequence keeps behind its first ones; some have fewer and keep them all."""
    r = random.Random(c["mix"] + 2)
    return [c["keep"] if i == 0 else int(c["keep"] * r.uniform(0.3, 1.2)) for i in range(c["n_seq"])]


def _starts(c):
    return [min(c["first"], n) for n in _lens(c)]


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


def _pool(gen, kind, pages, page, H, d, keys):
    x = _rows(gen, pages, page, H, d) if keys else torch.randn(pages, page, H, d, generator=gen, device="cuda")
    x = x.flatten(-2)[None]
    return _q8(x) if kind == "q8_0" else x.to(TORCH[kind])


def _prepare_evict(c, gen):
    """Gathered weights: a wide range, the first tokens far above the rest, some cells that no one ever saw."""
    L, n, H = c["L"], c["n_seq"], c["H"]
    lens = _lens(c)
    max_pages = -(-c["cells"] // c["page"])
    full = max_pages * c["page"]
    w = torch.empty(L, 2 * n, H, full, device="cuda")
    for l in range(L):
        x = torch.exp(1.5 * torch.randn(2 * n, H, full, generator=gen, device="cuda"))
        unseen = torch.rand(2 * n, 1, full, generator=gen, device="cuda") < 0.03
        w[l] = x.masked_fill_(unseen, 0.0)
        w[l, :, :, :4] *= 100.0
    L_idx = 1 if c.get("shared") else L
    n_idx = sum(min(k, m - s) for k, m, s in zip(_keeps(c), lens, _starts(c)))
    s = dict(weight=w, len=_ints(lens + [0] * n), src=_ints(list(range(n))), dst=_ints(list(range(n, 2 * n))),
             start=_ints(_starts(c)), keep=_ints(_keeps(c)), n_idx=n_idx, max_pages=max_pages,
             idx=torch.zeros(L_idx, n_idx, dtype=torch.int32, device="cuda"), cu=_ints([0] * (n + 1)),
             granted=_ints([0] * n), status=_ints([0] * n))
    # the cache's rows, which none of these calls reads: one page of them
    s["K"] = torch.zeros(L, 1, c["page"], H * 8, dtype=torch.float16, device="cuda")
    s["V"] = torch.zeros_like(s["K"])
    s["table"] = torch.full((2 * n, max_pages), -1, dtype=torch.int32, device="cuda")
    s["refs"] = _ints([0])
    return s


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=c)
    if c["entry"] == "evict":
        s.update(_prepare_evict(c, gen))
        torch.cuda.synchronize()
        return s
    lens = _lens(c)
    H, d, t, Hq = c["H"], c["d"], TORCH[c["type"]], c["H"] * c["G"]
    if c["entry"] == "prompt":
        n = c["n_tok"]
        k = _rows(gen, n, H, d)
        near = (torch.rand(n, generator=gen, device="cuda") * torch.arange(n, device="cuda")).long()
        q = 0.5 * k[near].repeat_interleave(c["G"], 1) + torch.randn(n, Hq, d, generator=gen, device="cuda")
        v = torch.randn(n, H, d, generator=gen, device="cuda")
        s.update(q=q.to(t), k=k.to(t), v=v.to(t), cu=_cu(lens), lens=lens,
                 o=torch.zeros(n, Hq, d, dtype=t, device="cuda"), lse=torch.zeros(n, Hq, device="cuda"))
        torch.cuda.synchronize()
        return s
    page, news = c["page"], _news(c)
    need = [-(-n // page) for n in lens]
    n_pages, max_pages = sum(need) + 3, max(need)
    order = torch.randperm(n_pages, generator=gen, device="cuda").cpu().numpy()
    table = np.full((c["n_seq"], max_pages), -1, np.int32)
    refs = np.zeros(n_pages, np.int32)
    refs[order[:sum(need)]] = 1
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        at += k
    n = sum(news)
    K = _pool(gen, c["cache"], n_pages, page, H, d, True)
    seen = (K if c["cache"] != "q8_0" else _q8_values(K)).reshape(-1, H, d)
    near = torch.randint(0, seen.shape[0], (n,), generator=gen, device="cuda")
    q = 0.5 * seen[near].float().repeat_interleave(c["G"], 1) + torch.randn(n, Hq, d, generator=gen, device="cuda")
    V = _pool(gen, c["cache"], n_pages, page, H, d, False) if c["entry"] == "cells" else torch.zeros_like(K)
    s.update(table=_ints(table), len=_ints(lens), refs=_ints(refs), K=K, V=V, q=q.to(t), cu=_cu(news), lens=lens,
             news=news, seqs=_ints(list(range(c["n_seq"]))), o=torch.zeros(n, Hq, d, dtype=t, device="cuda"),
             lse=torch.zeros(n, Hq, device="cuda"), bias=None, mask=None)
    if c.get("bias"):
        # beta = log of the fitted masses, a few of them at the fit's floor of 1e-12
        s["bias"] = torch.randn(1, n_pages, H, page, generator=gen, device="cuda")
        s["bias"].masked_fill_(torch.rand(s["bias"].shape, generator=gen, device="cuda") < 0.05, math.log(1e-12))
    if c.get("tree"):
        s["mask"] = torch.tensor(_tree_masks(c, news), dtype=torch.int64, device="cuda")
    if c["entry"] == "weigh":
        # log-sum-exps as the attention of these tokens left them, and what earlier tokens gathered
        s["weight"] = torch.exp(torch.randn(1, c["n_seq"], H, max_pages * page, generator=gen, device="cuda"))
        for i in range(c["n_seq"]):
            for x, seen, at in _scores(s, i):
                s["lse"][at] = torch.logsumexp(x.masked_fill_(~seen, NEG), -1).flatten(0, 1).t()
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------- the plain operators

def _softmax_rows(q, k, v, seen, bias, scale):
    """q [N][Hq][d], k and v [M][H][d], seen [N][M], bias [H][M] or None -> fp32 o [N][Hq][d], lse [N][Hq]."""
    N, Hq, d = q.shape
    M, H = k.shape[0], k.shape[1]
    G = Hq // H
    q = q.float().view(N, H, G, d).permute(1, 2, 0, 3).reshape(H, G * N, d)
    k = k.float().permute(1, 2, 0).contiguous()
    v = v.float().permute(1, 0, 2).contiguous()
    S = torch.bmm(q, k).mul_(scale).view(H, G, N, M)
    if bias is not None:
        S += bias[:, None, None, :]
    S.masked_fill_(~seen, NEG)
    m = S.amax(-1, keepdim=True)
    S = S.sub_(m.masked_fill(m == NEG, 0.0)).exp_()
    l = S.sum(-1, keepdim=True)
    o = torch.bmm(S.view(H, G * N, M), v).view(H, G, N, d) / torch.where(l > 0, l, 1.0)
    lse = (m + l.log()).view(H, G, N)
    return o.permute(2, 0, 1, 3).reshape(N, Hq, d), lse.permute(2, 0, 1).reshape(N, Hq)


def _plain_prompt(s):
    c = s["case"]
    first, last, step = c["first"], c["last"], 512
    at = 0
    for n in s["lens"]:
        for a in range(0, n, step):
            b = min(a + step, n)
            lo = max(min(first, b), a - last + 1)
            j = torch.cat([torch.arange(min(first, b), device="cuda"), torch.arange(lo, b, device="cuda")])
            i = torch.arange(a, b, device="cuda")[:, None]
            seen = (j <= i) & ((j < first) | (i - j < last))
            o, lse = _softmax_rows(s["q"][at + a:at + b], s["k"][at + j], s["v"][at + j], seen, None,
                                   1.0 / math.sqrt(c["d"]))
            s["o"][at + a:at + b] = o
            s["lse"][at + a:at + b] = lse
        at += n
    return dict(o=s["o"], lse=s["lse"])


def _cells(s, i, j):
    """Places of cells j of sequence i in the pool's rows."""
    page = s["case"]["page"]
    return s["table"][i].long()[j // page] * page + j % page


def _values(s, pool, at):
    c = s["case"]
    x = pool[0].reshape(-1, pool.shape[-1])[at]
    return (_q8_values(x) if c["cache"] == "q8_0" else x.float()).view(len(at), c["H"], c["d"])


def _bias(s, at):
    if s["bias"] is None:
        return None
    H = s["case"]["H"]
    return s["bias"][0].permute(0, 2, 1).reshape(-1, H)[at].t().contiguous()


def _seen(s, i, j, rows):
    """Which cells j of sequence i its tokens `rows` see: [rows][j]."""
    c = s["case"]
    first, last = c.get("first", 0), c.get("last", NO_WINDOW)
    base = s["lens"][i] - s["news"][i]
    t = torch.arange(rows.start, rows.stop, device="cuda")[:, None]
    if s["mask"] is None:
        return (j <= base + t) & ((j < first) | (base + t - j < last))
    at = sum(s["news"][:i])
    bits = s["mask"][at + rows.start:at + rows.stop, None]
    count = ((bits >> torch.arange(64, device="cuda")) & 1).sum(1, keepdim=True)
    drafted = ((bits >> (j - base).clamp(0, 63)) & 1) == 1
    return torch.where(j >= base, drafted & (j - base < 64), (j < first) | (j >= base - (last - count).clamp_min(0)))


def _plain_cells(s):
    c = s["case"]
    at = 0
    for i, (n, new) in enumerate(zip(s["lens"], s["news"])):
        lo = max(min(c["first"], n), n - new - c["last"] + 1)
        j = torch.cat([torch.arange(min(c["first"], n), device="cuda"), torch.arange(max(lo, 0), n, device="cuda")])
        p = _cells(s, i, j)
        o, lse = _softmax_rows(s["q"][at:at + new], _values(s, s["K"], p), _values(s, s["V"], p),
                               _seen(s, i, j, range(0, new)), _bias(s, p), 1.0 / math.sqrt(c["d"]))
        s["o"][at:at + new] = o
        s["lse"][at:at + new] = lse
        at += new
    return dict(o=s["o"], lse=s["lse"])


def _scores(s, i):
    """Scores of the counted tokens of sequence i over its cells, some tokens at a time:
    ([H][G][N][M] fp32, seen [N][M], the tokens' places)."""
    c = s["case"]
    n, new, H, G, d = s["lens"][i], s["news"][i], c["H"], c["G"], c["d"]
    j = torch.arange(n, device="cuda")
    p = _cells(s, i, j)
    k = _values(s, s["K"], p).permute(1, 2, 0).contiguous()
    b = _bias(s, p)
    at = sum(s["news"][:i])
    step = max(1, (1 << 28) // (n * H * G))
    for a in range(max(0, new - c.get("tail", new)), new, step):
        e = min(a + step, new)
        q = s["q"][at + a:at + e].float().view(e - a, H, G, d).permute(1, 2, 0, 3).reshape(H, -1, d)
        x = torch.bmm(q, k).mul_(1.0 / math.sqrt(d)).view(H, G, e - a, n)
        if b is not None:
            x += b[:, None, None, :]
        yield x, _seen(s, i, j, range(a, e)), slice(at + a, at + e)


def _plain_weigh(s):
    c = s["case"]
    for i, (n, new) in enumerate(zip(s["lens"], s["news"])):
        w = torch.zeros(c["H"], n, device="cuda")
        for x, seen, at in _scores(s, i):
            lse = s["lse"][at].t().reshape(c["H"], c["G"], -1, 1)
            w += x.sub_(lse).exp_().masked_fill_(~seen, 0.0).sum((1, 2))
        row = s["weight"][0, i]
        if c["decay"]:
            w[:, :n - new] += c["decay"] * row[:, :n - new]
        row[:, :n] = w
    return dict(weight=s["weight"])


def _plain_evict(s):
    c = s["case"]
    L, H, n = c["L"], c["H"], c["n_seq"]
    src, dst, start = s["src"].long(), s["dst"].long(), s["start"].long()
    lens = s["len"][src].long()
    kept = torch.minimum(s["keep"].long(), lens - start)
    s["cu"][1:] = kept.cumsum(0).int()
    s["granted"].copy_(s["src"])
    s["status"].zero_()
    # a cell's score: its heads' (and where all layers share the cells, its layers') sum in 64 bits, or the largest
    w = s["weight"][:, :n]
    groups = [range(L)] if c.get("shared") else [[l] for l in range(L)]
    cell = torch.arange(w.shape[-1], device="cuda")
    where = torch.arange(s["n_idx"], device="cuda")
    request = torch.searchsorted(s["cu"][1:].long(), where, right=True)
    for g, layers in enumerate(groups):
        score = torch.zeros(n, w.shape[-1], dtype=torch.float64, device="cuda")
        if c.get("most"):
            score.fill_(NEG)
        for l in layers:
            for h in range(H):
                x = w[l, :, h].double()
                score = torch.maximum(score, x) if c.get("most") else score + x
        score = score.float()
        score.masked_fill_(cell >= (lens - kept.clamp_max(c["recent"]))[:, None], float("inf"))
        score.masked_fill_((cell < start[:, None]) | (cell >= lens[:, None]), NEG)
        # the largest first, equal ones in the cells' order
        order = torch.sort(score, dim=1, descending=True, stable=True).indices
        rank = torch.empty_like(order).scatter_(1, order, cell.expand_as(order).contiguous())
        keep = rank < kept[:, None]
        at = torch.nonzero(keep)   # by request, cells ascending
        s["idx"][g, :len(at)] = (at[:, 1] - start[at[:, 0]]).int()
    to = start[request] + where - s["cu"].long()[request]
    for l in range(L):
        frm = start[request] + s["idx"][0 if c.get("shared") else l].long()
        s["weight"][l, dst[request], :, to] = s["weight"][l, src[request], :, frm]
        lead = cell < start[:, None]
        a = torch.nonzero(lead)
        s["weight"][l, dst[a[:, 0]], :, a[:, 1]] = s["weight"][l, src[a[:, 0]], :, a[:, 1]]
    return _evicted(s)


def _evicted(s):
    return {k: s[k] for k in ("idx", "cu", "granted", "status", "weight")}


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
    H = c["H"]
    if c["entry"] == "evict":
        n = c["n_seq"]
        cache = kc.KvCache(n_layers=c["L"], n_pages=1, page_size=c["page"], max_seqs=2 * n, max_pages=s["max_pages"],
                           n_head_kv=H, d_k=8, d_v=8, k_type=F16, v_type=F16, K=p(s["K"]), V=p(s["V"]), bias=None,
                           table=p(s["table"]), len=p(s["len"]), refs=p(s["refs"]))
        a = kc.PickArgs(seqs=p(s["src"]), start=p(s["start"]), keep=p(s["keep"]), weight=p(s["weight"]), idx=p(s["idx"]),
                        ld_idx=0 if c.get("shared") else s["n_idx"], cu=p(s["cu"]), granted=p(s["granted"]),
                        status=p(s["status"]), n_idx=s["n_idx"], recent=c["recent"],
                        heads=kc.HEADS_MAX if c.get("most") else kc.HEADS_SUM, max_len=c["cells"])
        need = dll.kvc_cache_pick_workspace(ctypes.byref(cache), n, ctypes.byref(a))
        return cache, a, None, torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    d, Hq = c["d"], H * c["G"]
    window = kc.Window(c["first"], c["last"]) if "last" in c else None
    if c["entry"] == "prompt":
        a = kc.PromptArgs(q=kc.Heads(p(s["q"]), Hq * d, d), k=kc.Heads(p(s["k"]), H * d, d),
                          v=kc.Heads(p(s["v"]), H * d, d), o=kc.Heads(p(s["o"]), Hq * d, d), lse=p(s["lse"]),
                          cu=p(s["cu"]), type=CODE[c["type"]], n_seq=c["n_seq"], n_tok=c["n_tok"], n_head=Hq,
                          n_head_kv=H, d_k=d, d_v=d)
        return a, window, None, None
    code = CODE[c["cache"]]
    cache = kc.KvCache(n_layers=1, n_pages=s["refs"].numel(), page_size=c["page"], max_seqs=s["len"].numel(),
                       max_pages=s["table"].shape[1], n_head_kv=H, d_k=d, d_v=d, k_type=code, v_type=code,
                       K=p(s["K"]), V=p(s["V"]), bias=p(s["bias"]), table=p(s["table"]), len=p(s["len"]),
                       refs=p(s["refs"]))
    a = kc.CacheAttnArgs(q=kc.Heads(p(s["q"]), Hq * d, d), o=kc.Heads(p(s["o"]), Hq * d, d), lse=p(s["lse"]),
                         seqs=p(s["seqs"]), cu=p(s["cu"]), mask=p(s["mask"]), mask_words=1, layer=0,
                         type=CODE[c["type"]], n_seq=c["n_seq"], n_tok=s["q"].shape[0], n_head=Hq,
                         max_new=max(s["news"]), max_len=max(s["lens"]))
    if c["entry"] == "weigh":
        x = kc.WeighArgs(weight=p(s["weight"]), decay=c["decay"], tail=c.get("tail", 0), fresh=0)
        return cache, a, window, x
    need = dll.kvc_attn_cache_window_workspace(ctypes.byref(cache), ctypes.byref(a), ctypes.byref(window))
    return cache, a, window, torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")


def _ok(rc, what):
    if rc:
        raise RuntimeError("%s returned %d" % (what, rc))


def _own(s):
    kc, dll = _library()
    if "calls" not in s:
        s["calls"] = _calls(s)
    c, (x, a, b, y) = s["case"], s["calls"]
    st = torch.cuda.current_stream().cuda_stream
    if c["entry"] == "prompt":
        _ok(dll.kvc_attn_prompt_window(x, a, st), "kvc_attn_prompt_window")
        return dict(o=s["o"], lse=s["lse"])
    if c["entry"] == "cells":
        _ok(dll.kvc_attn_cache_window(x, a, b, y.data_ptr(), y.numel(), st), "kvc_attn_cache_window")
        return dict(o=s["o"], lse=s["lse"])
    if c["entry"] == "weigh":
        _ok(dll.kvc_cache_weigh(x, a, b, y, st), "kvc_cache_weigh")
        return dict(weight=s["weight"])
    n = c["n_seq"]
    _ok(dll.kvc_cache_pick(x, n, a, y.data_ptr(), y.numel(), st), "kvc_cache_pick")
    _ok(dll.kvc_cache_take_weights(x, n, a.seqs, s["dst"].data_ptr(), a.start, a.cu, a.n_idx, a.idx, a.ld_idx, a.status,
                                   a.weight, st), "kvc_cache_take_weights")
    return _evicted(s)


def run(state):
    if own:
        return _own(state)
    plain = dict(prompt=_plain_prompt, cells=_plain_cells, weigh=_plain_weigh, evict=_plain_evict)
    return plain[state["case"]["entry"]](state)


# -------------------------------------------------------------------- work

def _pairs(n, new, first, last):
    """Cells that the last `new` of n tokens see, all together, and those that any of them sees."""
    base = n - new
    seen = sum(min(base + i + 1, min(first, base + i + 1) + last) for i in range(new))
    return seen, min(n, first + last - 1 + new)


def work(case):
    c = case
    lens = _lens(c)
    size = {"f32": 4.0, "f16": 2.0, "bf16": 2.0, "q8_0": 34.0 / 32}
    if c["entry"] == "evict":
        kept = [min(k, n - a) for k, n, a in zip(_keeps(c), lens, _starts(c))]
        rows = c["L"] * c["H"]
        read = rows * sum(lens) + 0.0
        moved = 2.0 * rows * (sum(kept) + sum(_starts(c)))
        return dict(bytes=4.0 * (read + moved + sum(kept) * (1 if c.get("shared") else c["L"])), flops=read)
    H, d, Hq = c["H"], c["d"], c["H"] * c["G"]
    if c["entry"] == "prompt":
        n = c["n_tok"]
        seen = sum(_pairs(m, m, c["first"], c["last"])[0] for m in lens)
        return dict(bytes=size[c["type"]] * n * (2 * Hq + 2 * H) * d + 4.0 * n * Hq, flops=4.0 * d * Hq * seen)
    news = _news(c)
    pairs = [_pairs(n, k, c.get("first", 0), c.get("last", NO_WINDOW)) for n, k in zip(lens, news)]
    row = size[c["cache"]] * H * d + (4 * H if c.get("bias") else 0)
    if c["entry"] == "cells":
        q = sum(news) * Hq * (2 * size[c["type"]] * d + 4)
        return dict(bytes=sum(p[1] for p in pairs) * (row + size[c["cache"]] * H * d) + q,
                    flops=4.0 * d * Hq * sum(p[0] for p in pairs))
    tails = [min(k, c.get("tail", k)) for k in news]
    pairs = [_pairs(n, k, c.get("first", 0), c.get("last", NO_WINDOW)) for n, k in zip(lens, tails)]
    q = sum(tails) * Hq * (size[c["type"]] * d + 4)
    held = 4.0 * H * (sum(lens) + (sum(lens) - sum(news) if c["decay"] else 0))
    return dict(bytes=sum(p[1] for p in pairs) * row + q + held, flops=2.0 * d * Hq * sum(p[0] for p in pairs))


# ------------------------------------------------- 64-bit results for checking

def _see(c, i, base, first, last, bits, n):
    """Token i behind base cells, of n cells in all: a truth value per cell, on the host."""
    see = np.zeros(n, bool)
    if bits is None:
        p = base + i
        see[max(0, p - last + 1):p + 1] = True
        see[:min(first, p + 1)] = True
        return see
    see[base - min(base, max(0, last - bin(bits).count("1"))):base] = True
    see[:min(first, base)] = True
    for j in range(n - base):
        see[base + j] = j < 64 and bits >> j & 1
    return see


def _exact_head(q, k, v, seen, bias, scale):
    """One head: q [N][d], k and v [M][d] in 64 bits, seen [N][M] -> o, lse."""
    x = torch.matmul(q, k.t().contiguous()) * scale
    if bias is not None:
        x = x + bias
    x = torch.where(seen, x, NEG)
    lse = torch.logsumexp(x, 1)
    return torch.matmul(torch.exp(x - torch.where(lse == NEG, 0.0, lse)[:, None]), v), lse


def _exact_prompt(c, s, scale):
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["lse"].shape, NEG, dtype=torch.float64, device="cuda")
    at = 0
    for n in _lens(c):
        for a in range(0, n, 1024):
            b = min(a + 1024, n)
            far = max(0, a - c["last"] + 1)
            cells = sorted(set(range(min(c["first"], b))) | set(range(far, b)))
            j = torch.tensor(cells, device="cuda")
            i = torch.arange(a, b, device="cuda").view(-1, 1)
            hidden = (j > i) | ((j >= c["first"]) & (j <= i - c["last"]))
            for h in range(c["H"] * c["G"]):
                g = h // c["G"]
                o[at + a:at + b, h], lse[at + a:at + b, h] = _exact_head(
                    s["q"][at + a:at + b, h].double(), s["k"][at + j, g].double(), s["v"][at + j, g].double(), ~hidden,
                    None, scale)
        at += n
    return dict(o=o, lse=lse)


def _exact_sequences(c, s):
    """(sequence, first token, tokens, K and V [n][H][d] in 64 bits, bias [H][n] or None, seen [new][n]) of a cache."""
    table = s["table"].cpu().numpy()
    bits = [int(b) & ((1 << 64) - 1) for b in s["mask"].cpu()] if s["mask"] is not None else None
    at = 0
    for i, (n, new) in enumerate(zip(_lens(c), _news(c))):
        pages = torch.tensor(table[i, :-(-n // c["page"])], device="cuda").long()
        k, v = (s[x][0, pages].reshape(-1, s[x].shape[-1])[:n] for x in "KV")
        k, v = ((_q8_values(x, True) if c["cache"] == "q8_0" else x.double()).view(n, c["H"], c["d"]) for x in (k, v))
        b = s["bias"][0, pages].permute(1, 0, 2).reshape(c["H"], -1)[:, :n].double() if s["bias"] is not None else None
        see = np.stack([_see(c, t, n - new, c.get("first", 0), c.get("last", NO_WINDOW), bits and bits[at + t], n)
                        for t in range(new)])
        yield i, at, new, k, v, b, torch.tensor(see, device="cuda")
        at += new


def _exact_evict(c, s):
    L, H, n = c["L"], c["H"], c["n_seq"]
    lens, starts, keeps = _lens(c), _starts(c), _keeps(c)
    kept = [min(k, m - a) for k, m, a in zip(keeps, lens, starts)]
    cu = [0] + np.cumsum(kept).tolist()
    after = s["weight"].double()
    idx = np.zeros(tuple(s["idx"].shape), np.int32)
    for l in range(L):
        if l and c.get("shared"):
            continue
        w = s["weight"][:, :n] if c.get("shared") else s["weight"][l:l + 1, :n]
        w = w.double().permute(1, 0, 2, 3).flatten(1, 2)
        score = (w.amax(1) if c.get("most") else w.sum(1)).float().cpu().numpy()
        for i in range(n):
            cells = np.arange(starts[i], lens[i])
            x = score[i, starts[i]:lens[i]].copy()
            x[cells >= lens[i] - min(c["recent"], kept[i])] = np.inf
            idx[l, cu[i]:cu[i + 1]] = np.sort(np.lexsort((cells, -x))[:kept[i]])
    for l in range(L):
        pick = idx[0 if c.get("shared") else l]
        for i in range(n):
            frm = list(range(starts[i])) + [starts[i] + x for x in pick[cu[i]:cu[i + 1]].tolist()]
            after[l, n + i, :, :len(frm)] = s["weight"][l, i][:, torch.tensor(frm, device="cuda").long()].double()
    return dict(idx=_ints(idx), cu=_ints(cu), granted=_ints(list(range(n))), status=_ints([0] * n), weight=after)


def exact(case, seed):
    c = case
    if c["entry"] == "evict":
        return _exact_evict(c, prepare(c, seed))
    s = prepare(c, seed)
    scale = 1.0 / math.sqrt(c["d"])
    if c["entry"] == "prompt":
        return _exact_prompt(c, s, scale)
    G = c["G"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["lse"].shape, NEG, dtype=torch.float64, device="cuda")
    weight = s["weight"].double() if c["entry"] == "weigh" else None
    for i, at, new, k, v, b, seen in _exact_sequences(c, s):
        if weight is not None:
            n = seen.shape[1]
            weight[0, i, :, n - new:n] = 0.0
            weight[0, i, :, :n - new] *= c["decay"]
            seen[:max(0, new - c.get("tail", new))] = False
        for h in range(c["H"] * G):
            q, g = s["q"][at:at + new, h].double(), h // G
            if weight is None:
                o[at:at + new, h], lse[at:at + new, h] = _exact_head(q, k[:, g], v[:, g], seen,
                                                                     None if b is None else b[g], scale)
                continue
            x = torch.matmul(q, k[:, g].t().contiguous()) * scale
            if b is not None:
                x += b[g]
            x = torch.exp(x - s["lse"][at:at + new, h].double()[:, None])
            weight[0, i, g, :seen.shape[1]] += torch.where(seen, x, 0.0).sum(0)
    return dict(weight=weight) if weight is not None else dict(o=o, lse=lse)
