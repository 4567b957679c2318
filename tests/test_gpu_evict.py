"""kvc_cache_pick and kvc_cache_take_weights (include/kvc-cache.h) against plain models: which cells are kept, in which
order, which requests are refused, and where their weights go."""
from __future__ import annotations

import numpy as np
import pytest

from kvc_harness import kc
from test_gpu_cache_attn import dev, dll   # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


def cache_of(L, seqs, max_pages, page, H, lens):
    """A cache whose rows no call here reads."""
    rows, table = dev(np.zeros(4096, np.uint8)), dev(np.full((seqs, max_pages), -1, np.int32))
    length, refs = dev(np.int32(lens)), dev(np.zeros(1, np.int32))
    c = kc.KvCache(n_layers=L, n_pages=1, page_size=page, max_seqs=seqs, max_pages=max_pages, n_head_kv=H, d_k=1, d_v=1,
                   k_type=kc.KV_TYPE_F32, v_type=kc.KV_TYPE_F32, K=rows.value, V=rows.value, table=table.value,
                   len=length.value, refs=refs.value)
    return c, (rows, table, length, refs)


def scores(w, most):
    """fp32 scores [cells] of weights [rows][cells], rows in order"""
    if most:
        out = np.full(w.shape[1], np.nan, np.float32)
        for x in w:
            out = np.fmax(out, x)
        return out
    s = np.zeros(w.shape[1])
    for x in w:
        s = s + x.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        return s.astype(np.float32)


def picked(score, start, n, keep, recent):
    """Indices from start of the kept cells."""
    k = min(keep, n - start)
    cells = np.arange(start, n)
    x = score[start:n].astype(np.float64)
    rank = np.where(np.isnan(x), -1, 0)                       # NaN below everything
    rank[cells >= n - min(recent, k)] = 1                     # the last ones above
    order = np.lexsort((cells, -np.where(np.isnan(x), 0, x), -rank))
    return np.sort(order[:k])


def model(w, lens, seqs, start, keep, recent, most, shared, n_idx, max_len, room):
    """(idx lists [layers][requests], cu, granted, status)"""
    L = w.shape[0]
    cu, granted, status, lists, seen = [0], [], [], [[] for _ in range(1 if shared else L)], []
    for i, s in enumerate(seqs):
        good = 0 <= s < len(lens) and s not in seen and 0 <= start[i] <= lens[s] <= min(max_len, room) and keep[i] >= 0
        seen.append(s)
        k = min(keep[i], lens[s] - start[i]) if good else 0
        if k > n_idx - cu[-1]:
            good, k = False, 0
        granted.append(s if good else -1)
        status.append(0 if good else kc.REQ_BAD)
        cu.append(cu[-1] + k)
        for g, out in enumerate(lists):
            if not good:
                out.append(np.zeros(0, np.int64))
                continue
            rows = w[:, s].reshape(-1, room) if shared else w[g, s]
            out.append(picked(scores(rows, most), start[i], lens[s], keep[i], recent))
    return lists, cu, granted, status


def run_pick(dll, w, lens, seqs, start, keep, recent, most=False, shared=False, n_idx=None, max_len=None, page=16, gap=0,   # noqa: F811
             runs=2):
    L, n_seqs, H, room = w.shape
    c, hold = cache_of(L, n_seqs, room // page, page, H, lens)
    n = len(seqs)
    max_len = max(lens) if max_len is None else max_len
    if n_idx is None:
        n_idx = model(w, lens, seqs, start, keep, recent, most, shared, 1 << 40, max_len, room)[1][-1]
    lists, cu, granted, status = model(w, lens, seqs, start, keep, recent, most, shared, n_idx, max_len, room)
    ld = 0 if shared else n_idx + gap
    idx = dev(np.full((L - 1) * ld + n_idx + 5, -7, np.int32))
    dw = dev(w)
    args = [dev(np.int32(x)) for x in (seqs, start, keep)]
    out = [dev(np.full(n + 1 + (x == 0), 99, np.int32)) for x in range(3)]   # cu, granted, status and one behind each
    a = kc.PickArgs(seqs=args[0].value, start=args[1].value, keep=args[2].value, weight=dw.value, idx=idx.value, ld_idx=ld,
                    cu=out[0].value, granted=out[1].value, status=out[2].value, n_idx=n_idx, recent=recent,
                    heads=kc.HEADS_MAX if most else kc.HEADS_SUM, max_len=max_len)
    size = dll.kvc_cache_pick_workspace(c, n, a)
    ws = dev(np.full(size + 16, 0xFF, np.uint8))
    what = f"pick L={L} H={H} lens={lens[:8]} seqs={seqs[:8]} start={start[:8]} keep={keep[:8]} recent={recent} most={most} shared={shared}"
    print(what, flush=True)
    for _ in range(runs):
        assert dll.kvc_cache_pick(c, n, a, ws.value, size, None) == 0
        got = [x.download(np.int32, n + 1 + (j == 0)).tolist() for j, x in enumerate(out)]
        assert got == [cu + [99], granted + [99], status + [99]], what
        got = idx.download(np.int32, (L - 1) * ld + n_idx + 5)
        want = np.full(got.size, -7, np.int32)
        for g, per in enumerate(lists):
            for i, x in enumerate(per):
                want[g * ld + cu[i]:g * ld + cu[i + 1]] = x
        assert np.array_equal(got, want), f"{what}: at {np.argwhere(got != want)[:5].ravel().tolist()}"
    assert (ws.download(np.uint8, 16, size) == 0xFF).all()
    assert np.array_equal(dw.download(np.uint32, w.size), w.view(np.uint32).ravel())
    if size:
        assert dll.kvc_cache_pick(c, n, a, ws.value, size - 1, None) == kc.E_SCRATCH
    return lists, cu


def random_weights(rng, L, seqs, H, room):
    w = np.exp(2 * rng.standard_normal((L, seqs, H, room))).astype(np.float32)
    w[:, :, :, rng.random(room) < 0.1] = 0
    return w


@pytest.mark.parametrize("most", [False, True])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("L,H", [(1, 1), (3, 2), (2, 8)])
def test_pick(dll, L, H, most, shared):   # noqa: F811
    rng = np.random.default_rng(L + H)
    lens = [300, 0, 1, 96, 17, 64]
    run_pick(dll, random_weights(rng, L, 6, H, 320), lens, [5, 0, 3, 1, 2, 4], [4, 0, 96, 0, 0, 16], [20, 150, 5, 3, 1, 1], 7, most, shared,
             gap=3)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 255, 256, 257, 1023, 1024, 1025, 1100, 4095, 4097])
def test_lengths(dll, n):   # noqa: F811
    rng = np.random.default_rng(n)
    w = random_weights(rng, 2, 1, 2, 4112)
    for keep in sorted({0, 1, 2, n // 5, n // 2, n - 1, n, n + 1, 1 << 30}):
        if keep >= 0:
            run_pick(dll, w, [n], [0], [min(3, n)], [keep], 2, runs=1)


@pytest.mark.parametrize("n", [9000, 16384, 32768, 33000, 70001])
@pytest.mark.parametrize("most", [False, True])
def test_long_sequences(dll, n, most):   # noqa: F811
    rng = np.random.default_rng(n)
    run_pick(dll, random_weights(rng, 1, 2, 2, 70016), [n, n // 3], [0, 1], [4, 100], [n // 5, n // 4], 128, most)


def test_equal_scores(dll):   # noqa: F811
    # all equal, two values, zeros of both signs: the lower index is kept
    for n, keep in ((1500, 700), (40, 7), (33000, 9000)):
        room = -(-n // 16) * 16
        w = np.ones((1, 1, 1, room), np.float32)
        run_pick(dll, w, [n], [0], [0], [keep], 5)
        w[..., ::3] = 2
        run_pick(dll, w, [n], [0], [0], [keep], 5)
        w[:] = 0
        w[..., ::2] = -0.0
        run_pick(dll, w, [n], [0], [2], [keep], 0)


def test_scores_that_are_not_finite(dll):   # noqa: F811
    rng = np.random.default_rng(5)
    w = random_weights(rng, 2, 1, 3, 528)
    w[0, 0, 1, 5:40] = np.nan
    w[0, 0, 0, 60] = np.inf
    w[0, 0, :, 70] = np.nan
    w[1, 0, 0, 80:90] = -np.inf
    w[1, 0, 1, 85] = np.inf                       # (a sum of both: NaN)
    w[1, 0, :, 100:110] = np.float32(3e38)        # (a sum past the largest float)
    w[:, 0, :, 200:210] = -1.0
    w[:, 0, :, 515:525] = np.nan                  # (among the last: kept)
    w[:, 0, :, 300:310] = np.float32(1e-45)       # the smallest there are
    for keep in (30, 200, 460, 500, 515, 527):
        for most in (False, True):
            for shared in (False, True):
                run_pick(dll, w, [527], [0], [3], [keep], 8, most, shared, runs=1)


def test_close_scores(dll):   # noqa: F811
    # sums that differ in their last bits only; what 32-bit sums would lose
    rng = np.random.default_rng(6)
    w = np.float32(1) + rng.integers(0, 3, (2, 1, 8, 1024)).astype(np.float32) * np.float32(2.0 ** -23)
    run_pick(dll, w, [1000], [0], [0], [500], 1)
    w = np.zeros((1, 1, 4, 1024), np.float32)
    w[0, 0, 0], w[0, 0, 1], w[0, 0, 2] = 1e8, rng.random(1024), -1e8
    run_pick(dll, w, [1000], [0], [0], [500], 1)


def test_refused_requests(dll):   # noqa: F811
    rng = np.random.default_rng(7)
    w = random_weights(rng, 2, 6, 2, 96)
    lens = [90, 50, 96, 40, 0, 95]
    # bad numbers, a sequence named twice (also behind a refused naming), bad starts and counts, too long
    run_pick(dll, w, lens, [0, -1, 6, 0, 1, 1, 3, 5, 4, 2], [4, 0, 0, 0, 51, 0, -1, 0, 0, 0], [20, 5, 5, 9, 5, 9, 3, 10, 8, -1], 3, max_len=94)
    # too few places: those that still fit are done
    run_pick(dll, w, lens, [0, 1, 2, 3, 5], [0, 0, 0, 0, 0], [30, 40, 25, 30, 15], 3, n_idx=70)
    run_pick(dll, w, lens, [0, 1, 2, 3, 5], [0, 0, 0, 0, 0], [30, 40, 25, 30, 15], 3, n_idx=0)
    run_pick(dll, w, lens, [0, 1], [0, 0], [(1 << 31) - 1, (1 << 31) - 1], (1 << 31) - 1)
    # lengths that the cache cannot have
    run_pick(dll, w, [97, -3, 96, (1 << 31) - 1, 5, 9], [0, 1, 2, 3, 4], [0] * 5, [9] * 5, 3, max_len=(1 << 31) - 1)


def test_many_requests(dll):   # noqa: F811
    rng = np.random.default_rng(8)
    n = kc.CACHE_MAX_REQUESTS
    lens = rng.integers(0, 49, n)
    w = random_weights(rng, 2, n, 1, 48)
    run_pick(dll, w, lens.tolist(), rng.permutation(n).tolist(), [0] * n, rng.integers(0, 60, n).tolist(), 3)


# ---------------------------------------------------------- weights that follow

def run_take(dll, L, H, room, seqs, src, dst, start, cu, idx, shared=False, status=None, n_idx=None, lens=None, page=16, gap=0):   # noqa: F811
    """idx: [layers][n_idx] or None (cu None: whole sequences)."""
    rng = np.random.default_rng(room + len(src))
    w = rng.standard_normal((L, seqs, H, room)).astype(np.float32)
    lens = [0] * seqs if lens is None else lens
    c, hold = cache_of(L, seqs, room // page, page, H, lens)
    want = w.copy()
    n_idx = (idx.shape[1] if idx is not None else 0) if n_idx is None else n_idx
    for i in range(len(src)):
        a, b = src[i], dst[i]
        if not (0 <= a < seqs and 0 <= b < seqs) or (status and status[i]):
            continue
        if cu is None:
            if 0 <= lens[b] <= room:
                want[:, b, :, :lens[b]] = w[:, a, :, :lens[b]]
            continue
        k = cu[i + 1] - cu[i]
        if start[i] < 0 or cu[i] < 0 or k < 0 or cu[i + 1] > n_idx or start[i] + k > room:
            continue
        want[:, b, :, :start[i]] = w[:, a, :, :start[i]]
        for l in range(L):
            for j in range(k):
                x = int(idx[0 if shared else l, cu[i] + j])
                if x >= j and start[i] + x < room:
                    want[l, b, :, start[i] + j] = w[l, a, :, start[i] + x]
    dw = dev(w)
    di = None
    if idx is not None:
        wide = np.full((idx.shape[0], idx.shape[1] + gap), 1 << 30, np.int32)
        wide[:, :idx.shape[1]] = idx
        di = dev(wide)
    ptr = [dev(np.int32(x)) if x is not None else None for x in (src, dst, start, cu, status)]
    val = [x.value if x is not None else None for x in ptr]
    print(f"take L={L} H={H} room={room} src={src[:8]} dst={dst[:8]} start={start and start[:8]} cu={cu and cu[:8]}", flush=True)
    assert dll.kvc_cache_take_weights(c, len(src), val[0], val[1], val[2], val[3], n_idx, di.value if di else None,
                                      0 if shared or idx is None else idx.shape[1] + gap, val[4], dw.value, None) == 0
    got = dw.download(np.float32, w.size).reshape(w.shape)
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32)), np.argwhere(got != want)[:5].tolist()


def ascending(rng, L, counts, n):
    return np.concatenate([np.stack([np.sort(rng.choice(n, k, replace=False)) for _ in range(L)]) for k in counts], 1).astype(np.int32)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("L,H,n", [(1, 1, 40), (3, 2, 500), (2, 5, 5000)])
def test_take(dll, L, H, n, shared):   # noqa: F811
    rng = np.random.default_rng(n)
    counts = [n // 3, 0, n, 1]
    idx = ascending(rng, 1 if shared else L, counts, n)
    cu = [0] + np.cumsum(counts).tolist()
    room = -(-(n + 20) // 16) * 16
    for src, dst in (([0, 1, 2, 3], [4, 5, 6, 7]), ([0, 1, 2, 3], [0, 1, 2, 3]), ([0, 0, 0, 2], [4, 5, 0, 7])):
        run_take(dll, L, H, room, 8, src, dst, [4, 7, 0, 9], cu, idx, shared, gap=5 * (not shared))


def test_take_after_a_fork(dll):   # noqa: F811
    run_take(dll, 2, 3, 96, 6, [0, 1, 1, 9, 2], [3, 4, 5, 2, -1], None, None, None, lens=[7, 90, 3, 7, 90, 96])
    run_take(dll, 2, 3, 96, 6, [0, 1], [3, 4], None, None, None, lens=[7, 90, 3, -4, 97, 96])
    run_take(dll, 2, 3, 96, 6, [0, 1], [3, 4], None, None, None, lens=[7, 90, 3, 9, 17, 96], status=[0, -2])


def test_take_refused(dll):   # noqa: F811
    rng = np.random.default_rng(1)
    idx = ascending(rng, 2, [10, 20, 30], 60)
    idx[0, 3], idx[1, 25], idx[0, 40], idx[1, 50] = 1, -5, 1 << 30, 95   # before their places, past the array
    for cu, start in (([0, 10, 30, 60], [0, 4, 9]), ([0, 10, 30, 61], [0, 4, 9]), ([-1, 10, 5, 60], [0, 0, 0]), ([0, 10, 30, 60], [-1, 90, 60]),
                      ([0, 10, 30, 60], [1 << 30, (1 << 31) - 1, 66])):
        run_take(dll, 2, 2, 96, 4, [0, 1, 2], [0, 1, 3], start, cu, idx)
        run_take(dll, 2, 2, 96, 4, [0, 1, 7], [0, -1, 3], start, cu, idx, status=[0, 3, kc.REQ_BAD])
    run_take(dll, 2, 2, 96, 4, [0, 1], [2, 3], [5, 9], [0, 0, 0], None)   # cut: the first ones only


def test_many_rows(dll):   # noqa: F811
    rng = np.random.default_rng(2)
    counts = rng.integers(0, 17, 700).tolist()
    run_take(dll, 4, 2, 16, 700, list(range(700)), list(range(700)), [0] * 700,
             [0] + np.cumsum(counts).tolist(), ascending(rng, 4, counts, 16))
