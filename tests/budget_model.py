"""Plain models, in numpy, of what keeps a cache to a budget (include/kvc-cache.h): which cells a sliding window shows,
and a paged cache of random rows with garbage wherever no sequence looks."""
from __future__ import annotations

import ctypes

import numpy as np

import kvcompact as kc
from cache_model import PagedModel, decode, encode


def window_seen(n, new, first, last, see=None):
    """Cells that the last `new` of n tokens see, [new][n]. see [new][new]: a tree's masks, whose drafted cells count as
    the last; None: each token sees those up to its own. last None: no window."""
    base = n - new
    out = np.zeros((new, n), bool)
    for i in range(new):
        if see is None:
            far = 0 if last is None else max(0, base + i + 1 - last)
            out[i, far:base + i + 1] = True
            if last is not None:
                out[i, :min(first, base + i + 1)] = True
        else:
            drafts = int(see[i].sum())
            far = 0 if last is None else max(0, base - max(0, last - drafts))
            out[i, far:base] = True
            if last is not None:
                out[i, :min(first, base)] = True
            out[i, base:] = see[i]
    return out


class PagedCells:
    """One layer (the last of `layers`) of a paged cache that holds sequences of `lens` cells at places of its own."""

    def __init__(self, cache, lens, H, dk, dv, page=16, bias=False, seed=0, layers=2, seqs=None, spare=2, edit=None,
                 bad_pages=()):
        from test_gpu_cache_attn import dev
        rng = self.rng = np.random.default_rng(seed)
        self.lens, self.H, self.layer, n_seq = lens, H, layers - 1, len(lens)
        max_pages = max(1, max(-(-m // page) for m in lens)) + 1
        n_pages = sum(-(-m // page) for m in lens) + 2
        m = self.m = PagedModel(layers, n_pages, page, n_seq + spare, max_pages, H, dk, dv, cache, cache, bias)
        order, at = rng.permutation(n_pages), 0
        self.place = rng.permutation(n_seq + spare)[:n_seq] if seqs is None else np.asarray(seqs)
        self.good = [0 <= s < n_seq + spare for s in self.place]
        for s, n, g in zip(self.place, lens, self.good):
            if not g:
                continue
            p = -(-n // page)
            m.table[s, :p] = order[at:at + p]
            m.len[s] = n
            at += p
        k = rng.standard_normal((n_pages, page, H, dk)) * np.exp(0.5 * rng.standard_normal((H, dk)))
        v = rng.standard_normal((n_pages, page, H, dv))
        if bias:
            m.bias[:] = rng.standard_normal(m.bias.shape) * 2

        def cell(s, j):
            """(page, cell) of cell j of sequence s of the call"""
            return m.table[self.place[s], j // page], j % page
        self.cell = cell
        if edit:
            edit(k, v, m.bias[self.layer] if bias else None, cell)
        with np.errstate(over="ignore", invalid="ignore"):
            m.K[self.layer] = encode(k.reshape(n_pages, page, -1), cache)
            m.V[self.layer] = encode(v.reshape(n_pages, page, -1), cache)
        used = np.zeros((n_pages, page), bool)
        for s in range(n_seq):
            if self.good[s]:
                for j in range(lens[s]):
                    used[cell(s, j)] = True
        m.K[self.layer][~used] = 0xFF
        m.V[self.layer][~used] = 0xFF
        if bias:
            m.bias[self.layer].transpose(0, 2, 1)[~used] = np.nan
        K, V = (decode(x[self.layer], cache).reshape(n_pages, page, H, -1) for x in (m.K, m.V))
        self.rows = []
        for s in range(n_seq):
            if not self.good[s]:
                self.rows.append(None)
                continue
            p, c = m.spots(m.table[self.place[s]].copy(), np.arange(lens[s]))
            b = m.bias[self.layer][p, :, c].T.astype(np.float64) if bias else None
            self.rows.append((K[p, c], V[p, c], b))
        self.hidden = [np.zeros(n, bool) for n in lens]
        for s, col, value in bad_pages:
            m.table[self.place[s], col] = value
            self.hidden[s][col * page:(col + 1) * page] = True
        self.bufs = {x: dev(getattr(m, x)) for x in ("K", "V", "table", "len", "refs")}
        if bias:
            self.bufs["bias"] = dev(m.bias)
        self.c = kc.KvCache(n_layers=layers, n_pages=n_pages, page_size=page, max_seqs=n_seq + spare, max_pages=max_pages,
                            n_head_kv=H, d_k=dk, d_v=dv, k_type=cache, v_type=cache,
                            **{x: y.value for x, y in self.bufs.items()})

    def ref(self):
        return ctypes.byref(self.c)
