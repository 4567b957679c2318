"""kvc_cache_weigh (include/kvc-cache.h): the softmax weight that tokens give each cell, against sums in 64 bits."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from budget_model import PagedCells, window_seen
from cache_model import BF16, F16, F32, Q8_0
from kvc_harness import kc
from test_gpu_cache_attn import KINDS, Strided, dev, dll, tree_masks, wide   # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


def weights_of(q, k, bias, seen, scale, lse, tail):
    """fp64 weights [H][M] of one sequence's tokens (q [N][Hq][d], k [M][H][d], lse [N][Hq] as given), and how far fp32
    sums of them may be off. With e = 2^-24, a pair's exponent is off by e (d + 8) |scale| sum |q||k| (the products'
    sum), 2 e (|s| + |bias| + |lse|) (the scale, the bias, the difference) and 2 e |x| (log2 e), its weight by as much
    and 4 e relative, and a sum of R weights by R e of it."""
    N, Hq, d = q.shape
    M, H = k.shape[0], k.shape[1]
    e = 2.0 ** -24
    w, tol = np.zeros((H, M)), np.zeros((H, M))
    for h in range(Hq):
        g = h // (Hq // H)
        for i in range(max(0, N - tail) if tail else 0, N):
            see = seen[i] if bias is None else seen[i] & (bias[g] != -np.inf)
            j = np.nonzero(see)[0]
            if not len(j) or np.isinf(lse[i, h]):   # (-inf: by definition; +inf: exp of -inf)
                continue
            s = (k[j, g] @ q[i, h]) * scale
            mag = (np.abs(k[j, g]) @ np.abs(q[i, h])) * abs(scale)
            b = bias[g, j] if bias is not None else np.zeros(len(j))
            x = s + b - lse[i, h]
            p = np.exp(x)
            w[g, j] += p
            with np.errstate(invalid="ignore"):
                off = e * (d + 8) * mag + 2 * e * (np.abs(s) + np.abs(b) + abs(lse[i, h])) + 2 * e * np.abs(x)
                tol[g, j] += p * (1.01 * off + 4 * e) + 2.0 ** -126
    return w, tol + (N * (Hq // H) + 4) * e * w


def log_sums(q, k, bias, seen, scale):
    """fp32 log-sum-exps as an attention would leave them [N][Hq]."""
    N, Hq, _ = q.shape
    H = k.shape[1]
    out = np.full((N, Hq), -np.inf)
    for h in range(Hq):
        g = h // (Hq // H)
        for i in range(N):
            see = seen[i] if bias is None else seen[i] & (bias[g] != -np.inf)
            if not see.any():
                continue
            s = (k[see, g] @ q[i, h]) * scale + (bias[g, see] if bias is not None else 0)
            m = s.max()
            out[i, h] = m + np.log(np.exp(s - m).sum()) if np.isfinite(m) else np.nan
    return out.astype(np.float32)


def run_weigh(dll, typ, cache, lens, news, H, G, d, page=16, bias=False, tree=False, words=1, window=None, decay=1.0, tail=0,   # noqa: F811
              fresh=0, seed=0, pad=0, shift=0, max_new=None, max_len=None, edit=None, bad_pages=(), seqs=None, empty=False,
              scale=0.0, runs=1, after=0, dv=None, lse_edit=None):
    p = PagedCells(cache, lens, H, d, dv or d, page, bias, seed, seqs=seqs, edit=edit, bad_pages=bad_pages)
    n_seq, Hq, n = len(lens), H * G, sum(news) + after
    cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    sq = Strided(p.rng.standard_normal((n, Hq, d)) * 1.2, typ, pad, shift)
    qd = wide(sq._view(sq.host), typ)
    room = p.m.max_pages * page
    old = np.exp(p.rng.standard_normal((p.layer + 1, n_seq + 2, H, room))).astype(np.float32)
    if decay == 0:
        old[:] = np.nan   # (not read)
    want, tol, written = old.astype(np.float64), np.zeros(old.shape), np.zeros(old.shape, bool)
    lse, masks = np.full((n, Hq), np.nan, np.float32), []
    first, last = window or (0, None)
    sc = scale or 1 / np.sqrt(d)
    for s in range(n_seq):
        nn, L = news[s], lens[s]
        bits, see = tree_masks(p.rng, nn, words, empty and nn > 0) if tree else (np.zeros((nn, 1), np.uint64), None)
        masks.append(bits)
        if not p.good[s] or nn > L or nn == 0:
            lse[cu[s]:cu[s + 1]] = -np.inf
            continue
        seen = window_seen(L, nn, first, last, see) & ~p.hidden[s]
        k, _, b = p.rows[s]
        x = slice(cu[s], cu[s + 1])
        with np.errstate(invalid="ignore", over="ignore"):
            lse[x] = log_sums(qd[x], k, b, seen, sc)
            if lse_edit:
                lse_edit(lse[x], s)
            w, t = weights_of(qd[x], k, b, seen, sc, lse[x].astype(np.float64), tail)
        at = (p.layer, p.place[s], slice(None), slice(0, L))
        had = want[at].copy()
        had[:, L - min(L, max(nn, fresh)):] = 0
        had = decay * had if decay else np.zeros_like(had)
        want[at], tol[at], written[at] = had + w, t + 2.0 ** -22 * had, True
    dl, dw = dev(lse), dev(old)
    extra = [dev(np.int32(p.place)), dev(cu), dev(np.concatenate(masks))]
    a = kc.CacheAttnArgs(q=sq.heads(), lse=dl.value, seqs=extra[0].value, cu=extra[1].value,
                         mask=extra[2].value if tree else None, mask_words=words if tree else 0, layer=p.layer, type=typ,
                         n_seq=n_seq, n_tok=n, n_head=Hq, max_new=max(news) if max_new is None else max_new,
                         max_len=max(lens) if max_len is None else max_len, scale=scale)
    x = kc.WeighArgs(dw.value, decay, tail, fresh)
    what = (f"weigh type={typ} cache={cache} lens={lens} news={news} H={H} G={G} d={d} page={page} bias={bias} tree={tree} "
            f"window={window} decay={decay} tail={tail} fresh={fresh}")
    print(what, flush=True)
    once = None
    for _ in range(runs):
        dw.upload(old)
        assert dll.kvc_cache_weigh(p.ref(), ctypes.byref(a), kc.Window(*window) if window else None, x, None) == 0
        got = dw.download(np.float32, old.size).reshape(old.shape)
        assert np.array_equal(got[~written].view(np.uint32), old[~written].view(np.uint32)), f"{what}: wrote elsewhere"
        assert np.array_equal(np.isnan(got[written]), np.isnan(want[written])), f"{what}: NaN"
        off = np.abs(got - want)
        ok = written & ~np.isnan(want)
        worst = (off[ok] / tol[ok].clip(1e-300)).max() if ok.any() else 0
        assert worst <= 1, f"{what}: {worst:.2f} times its bound at {np.argwhere(ok & (off > tol))[:4].tolist()}"
        once = got if once is None else once
        assert np.array_equal(once.view(np.uint32), got.view(np.uint32)), f"{what}: two runs differ"
    assert np.array_equal(dl.download(np.uint32, lse.size), lse.view(np.uint32).ravel())
    return got


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("bias", [False, True])
def test_single_tokens(dll, typ, cache, d, bias):   # noqa: F811
    run_weigh(dll, typ, cache, [1, 2, 33, 170, 64, 300], [1] * 6, 2, 4, d, bias=bias, seed=d, after=2, runs=2)


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [None, (0, 1), (4, 20), (40, 100), (0, 64), (1 << 30, 5)])
def test_trees(dll, typ, cache, d, window):   # noqa: F811
    run_weigh(dll, typ, cache, [300, 13, 64, 130], [13, 13, 5, 40], 2, 2, d, page=16 if d == 64 else 128, bias=d == 64, tree=True,
              window=window, decay=0.5, seed=d)


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [None, (4, 20), (33, 130), (0, 64)])
def test_prompts(dll, typ, cache, d, window):   # noqa: F811
    # all cells are those of the call's tokens; what the array held is not looked at
    run_weigh(dll, typ, cache, [290, 1, 64, 129], [290, 1, 64, 129], 1, 3, d, page=32, window=window, decay=0.0, seed=4)


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("tail", [1, 7, 32, 1000])
@pytest.mark.parametrize("window", [None, (4, 40)])
def test_last_tokens(dll, typ, cache, tail, window):   # noqa: F811
    run_weigh(dll, typ, cache, [290, 150, 64], [290, 40, 3], 1, 2, 128, page=32, bias=True, window=window, tail=tail, seed=5)
    run_weigh(dll, typ, cache, [290, 150, 64], [60, 40, 3], 1, 2, 64, page=32, bias=True, tree=True, window=window, tail=tail, seed=6)


@pytest.mark.parametrize("decay,fresh", [(0.0, 0), (1.0, 0), (0.9375, 5), (1.0, 1000), (0.0, 3)])
def test_decay_and_fresh_cells(dll, decay, fresh):   # noqa: F811
    run_weigh(dll, BF16, BF16, [200, 50, 9], [3, 1, 9], 2, 2, 64, decay=decay, fresh=fresh, seed=7)


@pytest.mark.parametrize("typ,cache", KINDS)
def test_larger_than_said(dll, typ, cache):   # noqa: F811
    for said in (0, 1, 1 << 20, (1 << 31) - 1):
        run_weigh(dll, typ, cache, [900, 120], [70, 3], 1, 2, 64, tree=True, words=2, seed=7, max_new=min(said, 1 << 20), max_len=said)


@pytest.mark.parametrize("words", [1, 2, 3])
def test_mask_words(dll, words):   # noqa: F811
    run_weigh(dll, BF16, BF16, [360, 150], [140, 65], 1, 2, 64, tree=True, words=words, seed=words)
    run_weigh(dll, BF16, BF16, [360, 150], [140, 65], 1, 2, 64, tree=True, words=words, seed=words, window=(3, 80))


@pytest.mark.parametrize("typ,cache", KINDS)
def test_sequences_that_have_no_part(dll, typ, cache):   # noqa: F811
    # a token whose mask is empty, more tokens than cells, bad sequence numbers, no tokens
    run_weigh(dll, typ, cache, [6, 4, 40, 9, 60, 30], [6, 5, 2, 3, 5, 0], 1, 2, 64, tree=True, seed=8, empty=True,
              seqs=[0, 3, -1, 77, 1, 2])


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("G", [2, 20])
def test_bias_that_hides(dll, typ, cache, G):   # noqa: F811
    def edit(k, v, b, cell):
        for j in range(20, 40):
            p, c = cell(0, j)
            b[p, :, c] = -np.inf
            k[p, c] = np.nan if cache != Q8_0 else 1.0
        for j in range(50):
            p, c = cell(1, j)
            b[p, 0, c] = -np.inf
    run_weigh(dll, typ, cache, [90, 50], [2, 1], 2, G, 64, bias=True, seed=9, edit=edit)


@pytest.mark.parametrize("typ,cache", [k for k in KINDS if k[1] != Q8_0])
@pytest.mark.parametrize("d", [64, 128, 256, 20])
@pytest.mark.parametrize("G", [2, 12])
def test_cells_that_are_not_finite(dll, typ, cache, d, G):   # noqa: F811
    # hidden cells gather nothing, whatever they hold; a NaN key makes the rows that see it NaN, and no other
    def edit(k, v, b, cell):
        for j in (6, 7, 30):
            p, c = cell(0, j)
            k[p, c] = np.nan
        p, c = cell(0, 97)
        k[p, c] = np.nan
    run_weigh(dll, typ, cache, [100], [12], 1, G, d, window=(3, 50), tree=True, seed=d, edit=edit)
    run_weigh(dll, typ, cache, [100], [1], 1, G, d, window=(3, 50), seed=d, edit=edit)


@pytest.mark.parametrize("typ,cache", KINDS)
def test_log_sums_as_given(dll, typ, cache):   # noqa: F811
    # -inf: nothing; +inf: nothing; rows of other sequences NaN
    def edit(lse, s):
        if s == 0:
            lse[1] = -np.inf
            lse[3, 0] = np.inf
            lse[5] += 2.5
    run_weigh(dll, typ, cache, [100, 40], [12, 3], 1, 2, 64, seed=10, lse_edit=edit)


@pytest.mark.parametrize("typ,cache", KINDS)
def test_bad_pages(dll, typ, cache):   # noqa: F811
    run_weigh(dll, typ, cache, [150, 80, 20], [3, 1, 2], 1, 2, 64, seed=10, bias=True,
              bad_pages=[(0, 1, 1 << 20), (0, 4, -1), (1, 0, -7), (2, 0, 1 << 30)])


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("d,dv,pad,shift", [(7, 9, 0, 0), (64, 64, 1, 0), (128, 64, 0, 1), (33, 250, 0, 0), (64, 128, 8, 8), (200, 8, 0, 0)])
def test_odd_heads_and_strides(dll, typ, d, dv, pad, shift):   # noqa: F811
    run_weigh(dll, typ, typ, [200, 45], [7, 1], 2, 2, d, dv=dv, bias=True, tree=True, seed=d, pad=pad, shift=shift, scale=0.2)
    run_weigh(dll, typ, typ, [100, 45], [90, 45], 1, 2, d, dv=dv, seed=d, pad=pad, shift=shift, scale=-0.1, decay=0.0)


@pytest.mark.parametrize("typ", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_q8_queries_of_any_alignment(dll, typ, d):   # noqa: F811
    run_weigh(dll, typ, Q8_0, [100, 45], [7, 1], 2, 3, d, bias=True, tree=True, seed=25, pad=1, shift=1)


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("G", [7, 40, 100])
def test_large_groups(dll, typ, cache, G):   # noqa: F811
    run_weigh(dll, typ, cache, [300, 20, 5], [1, 2, 3], 1, G, 64, tree=True, seed=G)


@pytest.mark.parametrize("typ,cache", [(F16, F16), (BF16, Q8_0)])
def test_many_sequences(dll, typ, cache):   # noqa: F811
    run_weigh(dll, typ, cache, [1 + 11 * i % 60 for i in range(150)], [1 + i % 2 if 1 + 11 * i % 60 > 1 else 1 for i in range(150)],
              1, 2, 64, seed=24, bias=True)


@pytest.mark.parametrize("typ", [F16, BF16])
@pytest.mark.parametrize("G", [1, 5, 33, 64, 65])
@pytest.mark.parametrize("announced", [None, 1 << 20])
def test_groups_of_many_rows(dll, typ, G, announced):   # noqa: F811
    # tiles of whole tokens with rows left over; four waves a block and (more cells announced: more blocks) eight
    run_weigh(dll, typ, typ, [300, 90], [140, 90], 1, G, 64, page=32, window=(5, 100) if G == 5 else None, decay=1.0, seed=G,
              max_len=announced)


@pytest.mark.parametrize("d", [32, 72, 96, 128, 136, 256])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("announced", [None, 1 << 20])
def test_head_widths_of_many_rows(dll, d, bias, announced):   # noqa: F811
    run_weigh(dll, BF16, BF16, [290, 77], [200, 77], 2, 2, d, page=16, bias=bias, window=(20, 150), decay=0.5, tail=0, seed=d,
              max_len=announced, runs=2)
    run_weigh(dll, F16, F16, [290, 200], [200, 150], 1, 2, d, page=16, bias=bias, tree=True, words=3, decay=1.0, tail=150, seed=d,
              max_len=announced)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("G", [1, 4])
def test_bad_cells_under_many_rows(dll, typ, G):   # noqa: F811
    # bad pages, keys that are not finite where nothing sees them, cells that the bias hides; one row and many
    def edit(k, v, b, cell):
        for j in (40, 41, 170):
            p, c = cell(0, j)
            k[p, c] = np.nan
            b[p, :, c] = -np.inf
    for news in ([1, 1], [200, 40]):
        run_weigh(dll, typ, typ, [400, 300], news, 2, G, 128, page=16, bias=True, seed=G, edit=edit, decay=0.5,
                  bad_pages=[(0, 4, -1), (0, 20, 1 << 30), (1, 0, -5)])
