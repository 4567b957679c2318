"""Attention with a sliding window and first tokens that stay visible
(include/kvc-cache.h, kvc_window), over prompts and over the paged cache, against
a 64-bit model with the error bounds of cache_model.attend."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from budget_model import PagedCells, window_seen
from cache_model import BF16, F16, F32, Q8_0, attend
from kvc_harness import kc
from test_gpu_cache_attn import KINDS, Strided, compare, dev, dll, join, tree_masks, typed, wide   # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu

WINDOWS = [(0, 1), (4, 16), (0, 64), (33, 40), (5, 100), (1000, 1), (0, 1 << 30), (1 << 30, 1 << 30), (64, 64)]


def run_prompt(dll, typ, lens, H, G, dk, dv, first, last, seed=0, pad=0, shift=0, tail=0, before=0, scale=0.0, edit=None,   # noqa: F811
               lse=True):
    rng = np.random.default_rng(seed)
    n, Hq = before + sum(lens) + tail, H * G
    k = rng.standard_normal((n, H, dk)) * np.exp(0.5 * rng.standard_normal((H, dk)))
    v = rng.standard_normal((n, H, dv))
    q = rng.standard_normal((n, Hq, dk)) + 0.5 * np.repeat(k, G, 1)
    if edit:
        edit(q, k, v)
    sq, sk, sv = (Strided(x, typ, pad, shift) for x in (q, k, v))
    so = Strided(np.full((n, Hq, dv), 7.0), typ, pad, shift)
    cu = before + np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    l, dcu = dev(np.full((n, Hq), 9.0, np.float32)), dev(cu)
    a = kc.PromptArgs(q=sq.heads(), k=sk.heads(), v=sv.heads(), o=so.heads(), lse=l.value if lse else None, cu=dcu.value,
                      type=typ, n_seq=len(lens), n_tok=n, n_head=Hq, n_head_kv=H, d_k=dk, d_v=dv, scale=scale)
    what = f"window prompt type={typ} lens={lens} H={H} G={G} dk={dk} dv={dv} first={first} last={last}"
    print(what, flush=True)
    assert dll.kvc_attn_prompt_window(ctypes.byref(a), kc.Window(first, last), None) == 0
    o, kept = so.read()
    assert kept, f"{what}: wrote between the rows"
    got_l = l.download(np.float32, n * Hq).reshape(n, Hq)
    q, k, v = (wide(s._view(s.host), typ) for s in (sq, sk, sv))
    parts = []
    with np.errstate(invalid="ignore"):
        for i, m in enumerate(lens):
            x = slice(cu[i], cu[i + 1])
            parts.append(attend(q[x], k[x], v[x], window_seen(m, m, first, last), None, scale or 1 / np.sqrt(dk), typ))
    want = join(parts, n, Hq, dv, cu)
    inside = slice(before, before + sum(lens))
    for x in (o, got_l):
        outside = np.concatenate([x[:before], x[before + sum(lens):]])
        fill = typed(np.full(1, 7.0), typ)[0] if x is o else 9.0
        assert (outside == fill).all(), f"{what}: wrote tokens of no sequence"
    if not lse:
        assert (got_l == 9.0).all()
        got_l = want[1].astype(np.float32)
    compare(o[inside], got_l[inside].astype(np.float64), tuple(w[inside] for w in want), typ, what)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("first,last", WINDOWS)
def test_prompt(dll, typ, d, first, last):   # noqa: F811
    run_prompt(dll, typ, [1, 0, 37, 64, 290], 1, 3, d, d, first, last, seed=d + last % 97)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("first,last", [(4, 70), (0, 200), (100, 64), (64, 129)])
def test_prompt_longer(dll, typ, first, last):   # noqa: F811
    # several row tiles whose tiles of keys begin at different places; tokens of no sequence around
    run_prompt(dll, typ, [500, 3, 430], 1, 2, 128, 128, first, last, seed=last, before=3, tail=5)


@pytest.mark.parametrize("typ", [F16, BF16])
@pytest.mark.parametrize("G", [1, 8])
def test_prompt_tile_edges(dll, typ, G):   # noqa: F811
    for first, last in ((0, 63), (0, 64), (0, 65), (63, 32), (64, 31), (65, 33), (128, 128)):
        run_prompt(dll, typ, [65, 127, 129, 257], 1, G, 64, 64, first, last, seed=G + last)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("dk,dv,pad,shift,scale", [(7, 9, 0, 0, 0.0), (40, 24, 0, 0, 0.0), (256, 3, 1, 0, 0.0), (64, 128, 8, 8, 0.3),
                                                   (64, 64, 0, 1, -0.1), (96, 96, 0, 0, -0.2), (200, 136, 0, 0, 0.0)])
def test_prompt_odd_heads_and_strides(dll, typ, dk, dv, pad, shift, scale):   # noqa: F811
    run_prompt(dll, typ, [150, 3, 41], 2, 2, dk, dv, 2, 50, seed=dk, pad=pad, shift=shift, scale=scale, lse=pad != 8)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("d", [64, 128, 256, 30])
def test_prompt_values_that_are_not_finite(dll, typ, d):   # noqa: F811
    # what a token holds reaches the rows whose window shows it, and no other: before, inside and behind the window
    def edit(q, k, v):
        v[1, :, 4] = np.inf           # one of the first: all later rows
        v[10, :, 5] = np.inf          # rows up to 49
        v[11, :, 5] = np.nan
        v[12, 0, 6] = -np.inf
        k[13] = np.nan
        v[200, :, 7] = -np.inf
        v[290:300] = np.nan           # (the next sequence)
        k[130, 0, 0] = np.inf
    run_prompt(dll, typ, [290, 10, 33], 1, 2, d, d, 3, 40, seed=d, edit=edit)
    run_prompt(dll, typ, [290, 10, 33], 1, 2, d, d, 0, 130, seed=d, edit=edit)


@pytest.mark.parametrize("typ", [F16, BF16])
def test_many_prompts(dll, typ):   # noqa: F811
    run_prompt(dll, typ, [(7 * i) % 5 * 17 for i in range(150)], 1, 2, 64, 64, 2, 30, seed=23, before=2, tail=3)


# ------------------------------------------------------------------ cells

def run_cells(dll, typ, cache, lens, news, H, G, dk, dv, first, last, page=16, bias=False, tree=False, words=1, seed=0, pad=0,   # noqa: F811
              shift=0, max_new=None, max_len=None, edit=None, bad_pages=(), seqs=None, empty=False, scale=0.0, runs=1, tail=0):
    p = PagedCells(cache, lens, H, dk, dv, page, bias, seed, seqs=seqs, edit=edit, bad_pages=bad_pages)
    n_seq, Hq, n = len(lens), H * G, sum(news) + tail
    q = p.rng.standard_normal((n, Hq, dk)) * 1.2
    cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    sq = Strided(q, typ, pad, shift)
    qd = wide(sq._view(sq.host), typ)
    parts, masks = [], []
    for s in range(n_seq):
        nn, L = news[s], lens[s]
        bits, see = tree_masks(p.rng, nn, words, empty) if tree else (np.zeros((nn, 1), np.uint64), None)
        masks.append(bits)
        if not p.good[s] or nn > L:
            parts.append((np.zeros((nn, Hq, dv)), np.full((nn, Hq), -np.inf), np.full((nn, Hq, dv), 1e-30), np.zeros((nn, Hq))))
            continue
        seen = window_seen(L, nn, first, last, see) & ~p.hidden[s]
        k, v, b = p.rows[s]
        with np.errstate(invalid="ignore"):
            parts.append(attend(qd[cu[s]:cu[s + 1]], k, v, seen, b, scale or 1 / np.sqrt(dk), typ))
    want = join(parts, n, Hq, dv, cu)
    so = Strided(np.full((n, Hq, dv), 7.0), typ, pad, shift)
    lse = dev(np.full((n, Hq), 9.0, np.float32))
    extra = [dev(np.int32(p.place)), dev(cu), dev(np.concatenate(masks))]
    a = kc.CacheAttnArgs(q=sq.heads(), o=so.heads(), lse=lse.value, seqs=extra[0].value, cu=extra[1].value,
                         mask=extra[2].value if tree else None, mask_words=words if tree else 0, layer=p.layer, type=typ,
                         n_seq=n_seq, n_tok=n, n_head=Hq, max_new=max(news) if max_new is None else max_new,
                         max_len=max(lens) if max_len is None else max_len, scale=scale)
    w = kc.Window(first, last)
    size = dll.kvc_attn_cache_window_workspace(p.ref(), ctypes.byref(a), w)
    ws = dev(np.full(max(size, 16), 0xFF, np.uint8))
    what = (f"window cells type={typ} cache={cache} lens={lens} news={news} H={H} G={G} dk={dk} dv={dv} page={page} bias={bias} "
            f"tree={tree} first={first} last={last} ws={size}")
    print(what, flush=True)
    e, once = sum(news), None
    for _ in range(runs):
        assert dll.kvc_attn_cache_window(p.ref(), ctypes.byref(a), w, ws.value, size, None) == 0
        o, kept = so.read()
        assert kept, f"{what}: wrote between the rows"
        l = lse.download(np.float32, n * Hq).reshape(n, Hq)
        assert (o[e:] == typed(np.full(1, 7.0), typ)[0]).all() and (l[e:] == 9.0).all(), f"{what}: wrote past the last sequence"
        compare(o[:e], l[:e].astype(np.float64), tuple(x[:e] for x in want), typ, what)
        once = o.copy() if once is None else once
        assert np.array_equal(once.view(np.uint8), o.view(np.uint8)), f"{what}: two runs differ"
    if size:
        assert dll.kvc_attn_cache_window(p.ref(), ctypes.byref(a), w, ws.value, size - 1, None) == kc.E_SCRATCH
        assert dll.kvc_attn_cache_window(p.ref(), ctypes.byref(a), w, None, size, None) == -1


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("first,last", WINDOWS)
def test_single_tokens(dll, typ, cache, d, first, last):   # noqa: F811
    run_cells(dll, typ, cache, [1, 2, 33, 170, 64, 400], [1, 1, 1, 1, 1, 1], 2, 4, d, d, first, last, bias=d == 64, seed=d, tail=2)


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("first,last", [(0, 1), (4, 20), (40, 64), (0, 200), (3, 9)])
def test_trees(dll, typ, cache, d, first, last):   # noqa: F811
    # windows shorter than a branch, as long as the drafts, longer
    run_cells(dll, typ, cache, [300, 13, 64, 330], [13, 13, 5, 40], 2, 2, d, d, first, last, page=16 if last != 64 else 128,
              bias=last == 20, tree=True, seed=d + last)


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("first,last", [(0, 1), (4, 20), (30, 130), (0, 64)])
def test_causal_chunks(dll, typ, cache, first, last):   # noqa: F811
    run_cells(dll, typ, cache, [400, 50, 31], [177, 50, 1], 1, 3, 128, 128, first, last, page=32, seed=4)


@pytest.mark.parametrize("typ,cache", KINDS)
def test_key_ranges(dll, typ, cache):   # noqa: F811
    # what is seen is long enough to be cut into ranges; the gap lies inside one, at its end, between two
    for first, last in ((4, 1500), (700, 1000), (512, 512), (600, 5)):
        run_cells(dll, typ, cache, [2300, 1, 900], [1, 1, 1], 1, 5, 128, 64 if cache != Q8_0 else 128, first, last, page=64,
                  bias=True, seed=5, runs=2)
    run_cells(dll, typ, cache, [2900, 90], [20, 9], 2, 1, 64, 64, 300, 600, page=16, tree=True, seed=6, runs=2)
    run_cells(dll, typ, cache, [2900, 90], [40, 9], 1, 2, 64, 64, 300, 600, page=16, tree=True, seed=7, runs=2)


@pytest.mark.parametrize("typ,cache", KINDS)
def test_larger_than_said(dll, typ, cache):   # noqa: F811
    run_cells(dll, typ, cache, [900, 120], [70, 3], 1, 2, 64, 64, 10, 300, tree=True, words=2, seed=7, max_new=1, max_len=1)
    run_cells(dll, typ, cache, [900, 120], [70, 3], 1, 2, 64, 64, 10, 300, seed=8, max_new=0, max_len=0)
    run_cells(dll, typ, cache, [900, 120], [70, 3], 1, 2, 64, 64, 10, 300, tree=True, words=2, seed=9, max_new=1 << 20,
              max_len=(1 << 31) - 1)


@pytest.mark.parametrize("words", [1, 2, 3])
def test_mask_words(dll, words):   # noqa: F811
    # (bits past mask_words * 64 are not there, and do not count)
    run_cells(dll, BF16, BF16, [360, 150], [140, 65], 1, 2, 64, 64, 3, 50, tree=True, words=words, seed=words)


def test_mask_bits_past_the_tokens(dll):   # noqa: F811
    """Bits of a mask at or past the number of new tokens name no cell, and count for nothing."""
    p = PagedCells(F16, [90], 1, 64, 64)
    q = Strided(p.rng.standard_normal((3, 2, 64)), F16)
    o, lse = Strided(np.zeros((3, 2, 64)), F16), dev(np.zeros((3, 2), np.float32))
    junk = 0xFFFFFFFFFFFFFFF8
    masks = np.array([[1 | junk, junk], [3 | junk, junk], [5 | junk, junk]], np.uint64)
    keep = [dev(np.int32(p.place)), dev(np.int32([0, 3])), dev(masks)]
    a = kc.CacheAttnArgs(q=q.heads(), o=o.heads(), lse=lse.value, seqs=keep[0].value, cu=keep[1].value, mask=keep[2].value,
                         mask_words=2, layer=p.layer, type=F16, n_seq=1, n_tok=3, n_head=2, max_new=3, max_len=90)
    assert dll.kvc_attn_cache_window(p.ref(), a, kc.Window(2, 10), None, 0, None) == 0
    see = np.array([[1, 0, 0], [1, 1, 0], [1, 0, 1]], bool)
    k, v, _ = p.rows[0]
    want = attend(wide(q._view(q.host), F16), k, v, window_seen(90, 3, 2, 10, see), None, 0.125, F16)
    compare(o.read()[0], lse.download(np.float32, 6).reshape(3, 2).astype(float), want, F16, "bits past the tokens")


@pytest.mark.parametrize("typ,cache", KINDS)
def test_rows_that_see_nothing(dll, typ, cache):   # noqa: F811
    run_cells(dll, typ, cache, [6, 4, 40, 9, 60], [6, 5, 2, 3, 5], 1, 2, 64, 64, 0, 1, tree=True, seed=8, empty=True,
              seqs=[0, 3, -1, 77, 1])


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("G", [2, 20])
def test_bias_that_hides(dll, typ, cache, G):   # noqa: F811
    low = np.finfo(np.float32).min

    def edit(k, v, b, cell):
        for j in range(60, 80):
            p, c = cell(0, j)
            b[p, :, c] = -np.inf
            k[p, c] = np.nan if cache != Q8_0 else 1.0
            v[p, c, :, ::3] = np.inf if cache != Q8_0 else 1.0
        for j in range(50):
            p, c = cell(1, j)
            b[p, 0, c] = -np.inf if j >= 30 or j < 2 else 3.0   # nothing that the window shows is left for head 0
            b[p, 1, c] = low if j >= 30 or j < 2 else 3.0       # nothing but the lowest for head 1
    run_cells(dll, typ, cache, [90, 50], [2, 1], 2, G, 64, 64, 2, 20, bias=True, seed=9, edit=edit)


@pytest.mark.parametrize("typ,cache", [k for k in KINDS if k[1] != Q8_0])
@pytest.mark.parametrize("d", [64, 128, 256, 20])
@pytest.mark.parametrize("G", [2, 12])
def test_cells_that_are_not_finite(dll, typ, cache, d, G):   # noqa: F811
    # in the gap they reach no row; at the window's edge only the rows that still see them; drafted, those of the branch
    def edit(k, v, b, cell):
        for j, x in ((1, np.inf), (6, np.nan), (40, np.nan), (41, np.inf), (70, np.inf), (72, np.nan), (91, np.inf),
                     (93, np.nan), (95, -np.inf)):
            p, c = cell(0, j)
            v[p, c, :, 3::5] = x
            if 6 <= j <= 41:
                k[p, c] = x
        p, c = cell(0, 97)
        k[p, c] = np.nan
    for tree in (False, True):
        run_cells(dll, typ, cache, [100], [12], 1, G, d, d, 3, 25, tree=tree, seed=d, edit=edit)
    run_cells(dll, typ, cache, [100], [1], 1, G, d, d, 3, 29, seed=d, edit=edit)


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("G", [1, 40])
def test_values_that_are_not_finite_in_a_long_range(dll, typ, cache, G):   # noqa: F811
    # more tiles than a block keeps apart, with the gap between them
    def edit(k, v, b, cell):
        for j, x, c in ((7, np.inf, 3), (2000, np.nan, 5), (2500, -np.inf, 7), (2503, np.inf, 7), (4990, np.nan, 9), (5005, -np.inf, 11)):
            p, i = cell(0, j)
            if cache == Q8_0:
                v[p, i, :, :32] *= 1e8
            else:
                v[p, i, :, c] = x
        for j in (9, 2501, 4995, 300, 3333, 2001):
            p, i = cell(0, j)
            b[p, :, i] = -np.inf
    run_cells(dll, typ, cache, [5010, 40], [2, 1], 2, G, 64, 64, 600, 2600, page=64, bias=True, tree=True, seed=43, edit=edit,
              max_len=1, runs=2)


@pytest.mark.parametrize("typ,cache", KINDS)
def test_bad_pages(dll, typ, cache):   # noqa: F811
    # bad page numbers in the gap, among the first cells, inside the window
    run_cells(dll, typ, cache, [350, 180, 20], [3, 1, 2], 1, 2, 64, 64, 40, 64, page=16, seed=10, bias=True,
              bad_pages=[(0, 1, 1 << 20), (0, 10, -1), (0, 19, -9), (1, 0, -7), (1, 5, 1 << 30), (2, 0, 1 << 30)])


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("dk,dv,pad,shift", [(7, 9, 0, 0), (64, 64, 1, 0), (128, 64, 0, 1), (33, 250, 0, 0), (64, 128, 8, 8)])
def test_odd_heads_and_strides(dll, typ, dk, dv, pad, shift):   # noqa: F811
    run_cells(dll, typ, typ, [200, 45], [7, 1], 2, 2, dk, dv, 4, 60, page=16, bias=True, tree=True, seed=dk, pad=pad,
              shift=shift, scale=0.2)


@pytest.mark.parametrize("typ", [F16, BF16])
@pytest.mark.parametrize("d,said", [(64, 17), (64, 40), (96, 40), (128, 40), (256, 17), (200, 40)])
def test_trees_of_several_row_tiles(dll, typ, d, said):   # noqa: F811
    run_cells(dll, typ, typ, [700, 290, 200], [140, 129, 3], 2, 2, d, d, 70, 200, page=32, bias=d != 96, tree=True, words=3,
              seed=d + said, max_new=said, max_len=200, runs=2)


@pytest.mark.parametrize("typ,cache", [(F16, F16), (BF16, Q8_0)])
def test_many_sequences(dll, typ, cache):   # noqa: F811
    run_cells(dll, typ, cache, [1 + 11 * i % 60 for i in range(150)], [1 + i % 2 if 1 + 11 * i % 60 > 1 else 1 for i in range(150)],
              1, 2, 64, 64, 2, 9, seed=24, bias=True)
