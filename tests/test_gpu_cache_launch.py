"""Launches of the cache's attention at the ends of what they are shaped for
(include/kvc-cache.h), and values that are not finite far apart."""
from __future__ import annotations

import numpy as np
import pytest

from cache_model import BF16, F16, F32, Q8_0, encode
from kvc_harness import kc
from test_gpu_cache_attn import dev, dll, run_cells, typed   # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ,cache", [(F32, F32), (BF16, BF16), (F16, Q8_0)])
@pytest.mark.parametrize("d", [64, 128])
def test_more_announced_than_a_launch_holds(dll, typ, cache, d):   # noqa: F811
    # 160 sequences of up to 2^20 new tokens would be more blocks than one launch takes
    lens = [70 + i % 30 if i % 40 == 0 else 3 + i % 5 for i in range(160)]
    news = [40 + i % 20 if i % 40 == 0 else 1 + i % 3 for i in range(160)]
    run_cells(dll, typ, cache, lens, news, 1, 2, d, d, tree=True, seed=40, max_new=1 << 20, max_len=1 << 20)


@pytest.mark.parametrize("typ,cache", [(F32, F32), (BF16, BF16), (F16, Q8_0)])
def test_longest_cache_announced(dll, typ, cache):   # noqa: F811
    for news in ([1, 1], [40, 9]):
        run_cells(dll, typ, cache, [300, 90], news, 1, 2, 64, 64, seed=41, max_len=(1 << 31) - 1, runs=2)


@pytest.mark.parametrize("typ,G", [(F16, 1), (F32, 1), (BF16, 40)])
def test_infinite_values_far_apart(dll, typ, G):   # noqa: F811
    """Two cells whose values are infinite, near the ends of long sequences whose key range is one block's, cost about
    what two of one tile cost: the cells between them are not gone through one by one. (A block that did would take
    hundreds of times longer; the bound leaves room for noise.)"""
    import hiprt
    H, d, page, cells, n_seq = 8, 64, 64, 4096, 512
    rng = np.random.default_rng(42)
    n_pages = cells // page
    t = typed(np.zeros(1), typ).dtype
    K, V = (typed(rng.standard_normal((n_pages * page, H, d)), typ) for _ in range(2))
    inf = typed(np.full(1, np.inf), typ)[0]
    bias = np.zeros((cells, H), np.float32)
    bias[5::97] = -np.inf                                       # (a hidden cell in every other tile or so)
    hidden = set(range(5, cells, 97))
    table = dev(np.tile(np.arange(n_pages, dtype=np.int32), (n_seq, 1)))
    length, refs = dev(np.full(n_seq, cells, np.int32)), dev(np.full(n_pages, n_seq, np.int32))
    cu, q = dev(np.arange(n_seq + 1, dtype=np.int32)), dev(typed(rng.standard_normal((n_seq, H * G, d)), typ))
    o, db = dev(np.zeros((n_seq, H * G, d), t)), dev(bias.reshape(n_pages, page, H).transpose(0, 2, 1))
    times, results = [], []
    for places in ((6, 7), (6, 3970)):
        v = V.copy()
        for p in places:
            assert p not in hidden and hidden & set(range(p // 32 * 32, p // 32 * 32 + 32))
            v[p, :, 3] = inf
        dk, dv = dev(K), dev(v)
        c = kc.KvCache(n_layers=1, n_pages=n_pages, page_size=page, max_seqs=n_seq, max_pages=n_pages, n_head_kv=H, d_k=d,
                       d_v=d, k_type=typ, v_type=typ, K=dk.value, V=dv.value, bias=db.value, table=table.value,
                       len=length.value, refs=refs.value)
        a = kc.CacheAttnArgs(q=kc.Heads(q.value, H * G * d, d), o=kc.Heads(o.value, H * G * d, d), cu=cu.value, type=typ,
                             n_seq=n_seq, n_tok=n_seq, n_head=H * G, max_new=1, max_len=cells)
        size = dll.kvc_attn_cache_workspace(c, a)
        ws = dev(np.zeros(max(size, 16), np.uint8))
        best = 1e9
        for _ in range(4):
            e0, e1 = hiprt.Event(), hiprt.Event()
            e0.record()
            assert dll.kvc_attn_cache(c, a, ws.value, size, None) == 0
            e1.record()
            best = min(best, e0.elapsed_ms(e1))
        times.append(best)
        results.append(o.download(t, n_seq * H * G * d).reshape(n_seq, H * G, d))
    print("one tile %.3f ms, far apart %.3f ms" % tuple(times), flush=True)
    for r in results:
        assert (r[..., 3] == inf).all()
    keep = [i for i in range(d) if i != 3]
    assert np.array_equal(results[0][..., keep], results[1][..., keep])
    assert times[1] < 8 * times[0] + 0.5


@pytest.mark.parametrize("typ,cache", [(F32, F32), (F16, F16), (BF16, BF16), (F16, Q8_0), (BF16, Q8_0)])
@pytest.mark.parametrize("G", [1, 40])
def test_values_that_are_not_finite_in_a_long_range(dll, typ, cache, G):   # noqa: F811
    # a range of more tiles than a block keeps apart: what is left out is added once, where it is seen
    def edit(q, k, v, b, cell):
        for j, x, c in ((7, np.inf, 3), (2500, -np.inf, 7), (2503, np.inf, 7), (4990, np.nan, 9), (5005, -np.inf, 11)):
            p, i = cell(0, j)
            if cache == Q8_0:
                v[p, i, :, :32] *= 1e8          # (a scale that is not finite)
            else:
                v[p, i, :, c] = x
        for j in (9, 2501, 4995, 300, 3333):
            p, i = cell(0, j)
            b[p, :, i] = -np.inf
        p, i = cell(0, 2505)
        b[p, 0, i] = -np.inf                    # hidden from one head, and not finite
        v[p, i, :, 13] = np.inf if cache != Q8_0 else 1.0
    run_cells(dll, typ, cache, [5010, 40], [2, 1], 2, G, 64, 64, page=64, bias=True, tree=True, seed=43, edit=edit, max_len=1,
              runs=2)


@pytest.mark.parametrize("typ,cache", [(F32, F32), (F16, F16), (BF16, Q8_0)])
@pytest.mark.parametrize("news,G", [([1, 1, 1], 2), ([20, 3, 9], 4), ([40, 1, 33], 4)])
def test_tokens_around_the_sequences(dll, typ, cache, news, G):   # noqa: F811
    # cu that begins behind 0 and ends before n_tok: the same results, bit for bit, and nothing else written
    H, d, page, lens = 2, 64, 32, [1500, 40, 333]
    rng = np.random.default_rng(44)
    pages = [-(-m // page) for m in lens]
    n_pages = sum(pages)
    K, V = (dev(encode(rng.standard_normal((n_pages * page, H * d)).astype(np.float32), cache)) for _ in range(2))
    table = np.full((3, max(pages)), -1, np.int32)
    for s, p in enumerate(pages):
        table[s, :p] = np.arange(p) + sum(pages[:s])
    held = [dev(x) for x in (table, np.int32(lens), np.ones(n_pages, np.int32))]
    c = kc.KvCache(n_layers=1, n_pages=n_pages, page_size=page, max_seqs=3, max_pages=max(pages), n_head_kv=H, d_k=d, d_v=d,
                   k_type=cache, v_type=cache, K=K.value, V=V.value, table=held[0].value, len=held[1].value, refs=held[2].value)
    n, Hq = sum(news), H * G
    q = typed(rng.standard_normal((n, Hq, d)), typ)
    out = []
    for before, after in ((0, 0), (3, 5)):
        m = before + n + after
        all_q = np.zeros((m, Hq, d), q.dtype)
        all_q[before:before + n] = q
        dq, o, lse = dev(all_q), dev(typed(np.full((m, Hq, d), 7.0), typ)), dev(np.full((m, Hq), 9.0, np.float32))
        cu = dev(np.int32(before + np.concatenate([[0], np.cumsum(news)])))
        h = [kc.Heads(x.value, Hq * d, d) for x in (dq, o)]
        a = kc.CacheAttnArgs(q=h[0], o=h[1], lse=lse.value, cu=cu.value, type=typ, n_seq=3, n_tok=m, n_head=Hq,
                             max_new=max(news), max_len=1500)
        size = dll.kvc_attn_cache_workspace(c, a)
        assert size > 0
        ws = dev(np.full(size, 0xFF, np.uint8))
        assert dll.kvc_attn_cache(c, a, ws.value, size, None) == 0
        x, l = o.download(q.dtype, m * Hq * d).reshape(m, Hq, d), lse.download(np.float32, m * Hq).reshape(m, Hq)
        rest = np.r_[0:before, before + n:m]
        assert (x[rest] == typed(np.full(1, 7.0), typ)[0]).all() and (l[rest] == 9.0).all()
        out.append((x[before:before + n].tobytes(), l[before:before + n].tobytes()))
    assert out[0] == out[1]
