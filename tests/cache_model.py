"""Plain models of the paged cache and of attention, in numpy, for the tests of
include/kvc-cache.h: the bookkeeping step by step on lists, rows as bytes, and
attention in 64 bits with the error its arithmetic may have."""
from __future__ import annotations

import numpy as np

import kvcompact as kc

BAD = kc.REQ_BAD
F32, F16, BF16, Q8_0 = kc.KV_TYPE_F32, kc.KV_TYPE_F16, kc.KV_TYPE_BF16, kc.KV_TYPE_Q8_0


def row_bytes(typ, n):
    return {F32: 4 * n, F16: 2 * n, BF16: 2 * n, Q8_0: n // 32 * 34}[typ]


def bf16(x):
    """fp32 -> bf16 bits, to nearest even (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def encode(x, typ):
    """fp32 [..., n] -> row bytes [..., row_bytes]; Q8_0 by kv_quantize_row's steps (scale cut to fp16)."""
    x = np.ascontiguousarray(x, np.float32)
    if typ == F32:
        return x.view(np.uint8)
    if typ == F16:
        return x.astype(np.float16).view(np.uint8)
    if typ == BF16:
        return bf16(x).view(np.uint8)
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(b).max(-1, keepdims=True)
    d = (amax / np.float32(127.0)).astype(np.float32)
    cut = (d.view(np.uint32) & np.uint32(0xFFFFE000)).view(np.float32).astype(np.float16)   # (normal scales)
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.where(d != 0, np.float32(127.0) / amax, np.float32(0)).astype(np.float32)
    v = np.clip((b * inv).astype(np.float32), -128, 127)
    q = (np.sign(v) * np.floor(np.abs(v).astype(np.float64) + 0.5)).astype(np.int8)
    return np.concatenate([cut.view(np.uint8), q.view(np.uint8)], -1).reshape(*x.shape[:-1], -1)


def decode(b, typ):
    """row bytes -> fp64 values."""
    b = np.ascontiguousarray(b)
    if typ == F32:
        return b.view(np.float32).astype(np.float64)
    if typ == F16:
        return b.view(np.float16).astype(np.float64)
    if typ == BF16:
        return (b.view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    b = b.reshape(*b.shape[:-1], -1, 34)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    return (d * np.ascontiguousarray(b[..., 2:]).view(np.int8)).reshape(*b.shape[:-2], -1)


class PagedModel:
    """The cache of include/kvc-cache.h on the host."""

    def __init__(self, L, pages, page, seqs, max_pages, H, dk, dv, k_type, v_type, bias):
        self.L, self.n_pages, self.page, self.max_seqs, self.max_pages = L, pages, page, seqs, max_pages
        self.H, self.dk, self.dv, self.k_type, self.v_type = H, dk, dv, k_type, v_type
        self.K = np.zeros((L, pages, page, row_bytes(k_type, H * dk)), np.uint8)
        self.V = np.zeros((L, pages, page, row_bytes(v_type, H * dv)), np.uint8)
        self.bias = np.zeros((L, pages, H, page), np.float32) if bias else None
        self.table = np.full((seqs, max_pages), -1, np.int32)
        self.len = np.zeros(seqs, np.int32)
        self.refs = np.zeros(pages, np.int32)

    def _pages(self, cells):
        return -(-cells // self.page)

    def spots(self, row, cells):
        """(page, cell) of cells through a table row."""
        cells = np.asarray(cells, np.int64)
        return np.asarray(row)[cells // self.page], cells % self.page

    def _requests(self, seqs):
        out, seen = [], set()
        for s in seqs:
            ok = 0 <= s < self.max_seqs and s not in seen
            if 0 <= s < self.max_seqs:
                seen.add(s)
            out.append(int(s) if ok else -1)
        return out

    def _grant(self, needs):
        """First free page of each request's share, all or none; the free pages; what is missing."""
        free = [p for p in range(self.n_pages) if self.refs[p] == 0]
        used, at, missing = 0, [], []
        for k in needs:
            m = 0
            if k < 0:
                a = -1
            elif used + k <= len(free):
                a, used = used, used + k
            else:
                a, m = -1, k - (len(free) - used)
            at.append(a)
            missing.append(m)
        return free, at, missing

    def extend(self, seqs, counts):
        ids = self._requests(seqs)
        refs0 = self.refs.copy()
        needs, plan = [], []
        for s, k in zip(ids, counts):
            need, copied = -1, False
            if s >= 0 and k >= 0 and self.len[s] + k <= self.max_pages * self.page:
                old = int(self.len[s])
                copied = bool(old % self.page and k and refs0[self.table[s, old // self.page]] > 1)
                need = self._pages(old + k) - self._pages(old) + copied
            needs.append(need)
            plan.append(copied)
        free, at, missing = self._grant(needs)
        status, copies = [], []
        for s, k, need, a, m, copied in zip(ids, counts, needs, at, missing, plan):
            if need < 0 or a < 0:
                status.append(m or BAD)
                continue
            status.append(0)
            old = int(self.len[s])
            first = self._pages(old) - copied
            if copied:
                copies.append((self.table[s, first], free[a], old % self.page))
                self.refs[self.table[s, first]] -= 1
            for j in range(need):
                self.table[s, first + j] = free[a + j]
                self.refs[free[a + j]] = 1
            self.len[s] = old + k
        for a, b, n in copies:
            self.K[:, b, :n] = self.K[:, a, :n]
            self.V[:, b, :n] = self.V[:, a, :n]
            if self.bias is not None:
                self.bias[:, b, :, :n] = self.bias[:, a, :, :n]
        return status

    def write(self, layer, n_layers, seqs, cu, K, V):
        """K, V: row bytes [n_layers][rows][...]."""
        for i, s in enumerate(seqs):
            n = cu[i + 1] - cu[i]
            if not 0 <= s < self.max_seqs:
                continue
            for r in range(n):
                cell = int(self.len[s]) - n + r
                if cell < 0:
                    continue
                p, c = self.table[s, cell // self.page], cell % self.page
                self.K[layer:layer + n_layers, p, c] = K[:, cu[i] + r]
                self.V[layer:layer + n_layers, p, c] = V[:, cu[i] + r]
                if self.bias is not None:
                    self.bias[layer:layer + n_layers, p, :, c] = 0

    def fork(self, src, dst):
        ids, len0 = self._requests(dst), self.len.copy()
        table0, status = self.table.copy(), []
        for a, s in zip(src, ids):
            if s < 0 or not 0 <= a < self.max_seqs or a == s or len0[s]:
                status.append(BAD)
                continue
            status.append(0)
            n = self._pages(int(len0[a]))
            self.table[s, :n] = table0[a, :n]
            for p in table0[a, :n]:
                self.refs[p] += 1
            self.len[s] = len0[a]
        return status

    def free(self, seqs):
        for s in self._requests(seqs):
            if s < 0:
                continue
            n = self._pages(int(self.len[s]))
            for p in self.table[s, :n]:
                self.refs[p] -= 1
            self.table[s, :n] = -1
            self.len[s] = 0

    def compact(self, seqs, start, cu, idx, values=None, beta=None):
        """idx [L][n_idx]; values: V row bytes [L][n_idx][...]; beta [L][H][n_idx]."""
        ids, refs0, table0 = self._requests(seqs), self.refs.copy(), self.table.copy()
        needs, plan = [], []
        for i, s in enumerate(ids):
            n = cu[i + 1] - cu[i]
            good = s >= 0 and 0 <= start[i] <= self.len[s] and 0 <= n <= self.len[s] - start[i]
            first = start[i] // self.page
            end = self._pages(start[i] + n) if good else 0
            shared = [j for j in range(first, end) if n and refs0[self.table[s, j]] > 1] if good else []
            needs.append(len(shared) if good else -1)
            plan.append((n, first, end, shared))
        free, at, missing = self._grant(needs)
        status = []
        jobs = []
        for i, s in enumerate(ids):
            if needs[i] < 0 or at[i] < 0:
                status.append(missing[i] or BAD)
                continue
            status.append(0)
            n, first, end, shared = plan[i]
            held = self._pages(int(self.len[s]))
            for k, j in enumerate(shared):
                self.refs[self.table[s, j]] -= 1
                self.table[s, j] = free[at[i] + k]
                self.refs[free[at[i] + k]] = 1
            for j in range(end, held):
                self.refs[self.table[s, j]] -= 1
                self.table[s, j] = -1
            self.len[s] = start[i] + n
            if n:
                jobs.append((i, s, n, first in shared))
        old = [x.copy() if x is not None else None for x in (self.K, self.V, self.bias)]
        for i, s, n, lead in jobs:
            cells = np.arange(start[i] // self.page * self.page, start[i]) if lead else np.zeros(0, np.int64)
            for l in range(self.L):
                frm = np.concatenate([cells, start[i] + idx[l][cu[i]:cu[i + 1]].astype(np.int64)])
                to = np.concatenate([cells, start[i] + np.arange(n)])
                (a, b), (c, d) = self.spots(table0[s], frm), self.spots(self.table[s], to)
                self.K[l, c, d] = old[0][l, a, b]
                self.V[l, c, d] = old[1][l, a, b]
                m = len(cells)
                if values is not None:
                    self.V[l, c[m:], d[m:]] = values[l][cu[i]:cu[i + 1]]
                if self.bias is not None:
                    self.bias[l, c, :, d] = old[2][l, a, :, b]
                    if beta is not None:
                        self.bias[l, c[m:], :, d[m:]] = beta[l][:, cu[i]:cu[i + 1]].T
        return status


def attend(q, k, v, seen, bias, scale, typ, split_kv=False):
    """fp64 attention of one sequence: q [N][Hq][dk], k [M][H][dk], v [M][H][dv], seen [N][M], bias [H][M] or None.

    Returns o, lse and how far each may be off. With u the half step of the type (2^-24, 2^-11, 2^-8) and e = 2^-24:
      a score is off by at most e (dk + 4) |scale| sum |q||k| (sums of dk products in fp32, the scale, the bias) and
      its weight's exponent by 2 e max |s - m|: together ds, so a weight by 2 ds + 4 e relative (exp and the
      running rescales; ds is small);
      weights are rounded by u (16-bit types; sums of M of them by M e), and the result by u.
    fp16 has a spacing of 2^-24 below 2^-14, so a result there is off by half of it, 2^-25, whatever its size, and a
    weight (held as 2^10 exp(s - m)) by 2^-35.
    """
    N, Hq, dk = q.shape
    M, H = k.shape[0], k.shape[1]
    e = 2.0 ** -24
    u = {F32: e, F16: 2.0 ** -11, BF16: 2.0 ** -8}[typ]
    low = 2.0 ** -25 if typ == F16 else 0.0
    o, lse = np.zeros((N, Hq, v.shape[2])), np.full((N, Hq), -np.inf)
    tol_o, tol_l = np.zeros_like(o), np.zeros_like(lse)
    for h in range(Hq):
        g = h // (Hq // H)
        for i in range(N):
            see = seen[i] if bias is None else seen[i] & (bias[g] != -np.inf)
            j = np.nonzero(see)[0]
            if not len(j):
                continue
            s = (k[j, g] @ q[i, h]) * scale
            mag = (np.abs(k[j, g]) @ np.abs(q[i, h])) * abs(scale)   # (a size: a negative scale has the same)
            if bias is not None:
                s = s + bias[g, j]
                mag = mag + np.abs(bias[g, j])
            m = s.max()
            if not m < np.inf:   # a NaN or +inf score: the whole row is NaN
                o[i, h], lse[i, h] = np.nan, np.nan
                continue
            w = np.exp(s - m)
            l = w.sum()
            o[i, h] = (w @ v[j, g]) / l
            lse[i, h] = m + np.log(l)
            wide = s - m > -40
            assert np.isfinite(mag[wide]).all()
            ds = e * (dk + 4) * mag[wide].max() + 2 * e * np.abs(s - m)[wide].max()
            rel = 2 * ds + (8 + len(j)) * e
            size = (w @ np.where(np.isfinite(v[j, g]), np.abs(v[j, g]), 0)) / l
            tol_o[i, h] = u * np.where(np.isfinite(o[i, h]), np.abs(o[i, h]), 0) + (0 if typ == F32 else u) * size * (1 + u) + 2 * rel * size + 1e-30
            tol_o[i, h] += low + low * 2.0 ** -10 * np.where(np.isfinite(v[j, g]), np.abs(v[j, g]), 0).sum(0) / l
            tol_l[i, h] = rel + 4 * e * (abs(m) + abs(lse[i, h]) + 1)
    return o, lse, tol_o, tol_l
