"""Attention over the paged cache and over whole prompts (include/kvc-cache.h)
against a 64-bit model, with the error bounds of cache_model.attend."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from cache_model import BF16, F16, F32, PagedModel, Q8_0, attend, bf16, decode, encode
from kvc_harness import kc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dll():
    lib = kc.load_product()
    if not lib.dll.kv_compact_hip_available():
        pytest.fail("no usable GPU for the GPU test tier")
    return kc.bind_cache(lib.dll)


def dev(x):
    import hiprt
    x = np.ascontiguousarray(x)
    b = hiprt.DevBuf(max(x.nbytes, 16))
    if x.nbytes:
        b.upload(x)
    return b


def typed(x, typ):
    """fp32 -> the type's array (bf16 as uint16)."""
    x = np.asarray(x, np.float32)
    return {F32: lambda: x, F16: lambda: x.astype(np.float16), BF16: lambda: bf16(x)}[typ]()


def wide(x, typ):
    """back to fp64"""
    return decode(np.ascontiguousarray(x).view(np.uint8).reshape(*x.shape[:-1], -1), typ)


class Strided:
    """[n][heads][d] of a type on the device, with gaps of `pad` elements behind tokens and heads and `shift` before."""

    def __init__(self, x, typ, pad=0, shift=0, fill=None):
        n, H, d = x.shape
        self.typ, self.n, self.H, self.d, self.pad, self.shift = typ, n, H, d, pad, shift
        host = np.full(shift + n * (H * (d + pad) + pad), 0, typed(np.zeros(1), typ).dtype)
        host[:] = typed(np.full(1, 3.0 if fill is None else fill), typ)
        view = self._view(host)
        view[:] = x if x.dtype == host.dtype else typed(x, typ)
        self.host, self.buf = host, dev(host)

    def _view(self, host):
        rows = host[self.shift:].reshape(self.n, -1)[:, :self.H * (self.d + self.pad)] if self.n else host[:0].reshape(0, self.H * (self.d + self.pad))
        return rows.reshape(self.n, self.H, self.d + self.pad)[:, :, :self.d]

    def heads(self):
        return kc.Heads(self.buf.value + self.shift * self.host.itemsize, self.H * (self.d + self.pad) + self.pad,
                        self.d + self.pad)

    def read(self):
        """values, and whether everything between them is as it was"""
        got = self.buf.download(self.host.dtype, self.host.size)
        a, b = got.copy(), self.host.copy()
        self._view(a)[:] = 0
        self._view(b)[:] = 0
        return self._view(got).copy(), np.array_equal(a.view(np.uint8), b.view(np.uint8))


def compare(o, lse, want, typ, what):
    ro, rl, to, tl = want
    o = wide(o, typ)
    assert np.array_equal(np.isnan(o), np.isnan(ro)), f"{what}: NaN"
    with np.errstate(invalid="ignore"):
        off = np.abs(o - ro)
        off[(o == ro) | np.isnan(ro)] = 0
        worst = (off / to.clip(1e-300)).max() if off.size else 0
    assert worst <= 1, f"{what}: o {worst:.2f} times its bound at {np.argwhere(off > to)[:4].tolist()}"
    with np.errstate(invalid="ignore"):
        dl = np.abs(lse - rl)
        dl[(lse == rl) | (np.isnan(lse) & np.isnan(rl))] = 0
    worst = (dl / tl.clip(1e-300)).max() if dl.size else 0
    assert worst <= 1, f"{what}: lse {worst:.2f} times its bound"


def join(parts, n_tok, Hq, dv, cu):
    out = (np.zeros((n_tok, Hq, dv)), np.zeros((n_tok, Hq)), np.zeros((n_tok, Hq, dv)), np.zeros((n_tok, Hq)))
    for i, p in enumerate(parts):
        for a, b in zip(out, p):
            a[cu[i]:cu[i + 1]] = b
    return out


# ---------------------------------------------------------------- prompts

def run_prompt(dll, typ, lens, H, G, dk, dv, seed=0, pad=0, shift=0, tail=0, first=0, lse=True, scale=0.0, edit=None):
    rng = np.random.default_rng(seed)
    n = first + sum(lens) + tail
    Hq = H * G
    k = rng.standard_normal((n, H, dk)) * np.exp(0.5 * rng.standard_normal((H, dk)))
    v = rng.standard_normal((n, H, dv))
    q = rng.standard_normal((n, Hq, dk)) + 0.5 * np.repeat(k, G, 1)
    if edit:
        edit(q, k, v)
    sq, sk, sv = (Strided(x, typ, pad, shift) for x in (q, k, v))
    so = Strided(np.full((n, Hq, dv), 7.0), typ, pad, shift)
    cu = first + np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    l = dev(np.full((n, Hq), 9.0, np.float32))
    dcu = dev(cu)
    a = kc.PromptArgs(q=sq.heads(), k=sk.heads(), v=sv.heads(), o=so.heads(), lse=l.value if lse else None, cu=dcu.value,
                      type=typ, n_seq=len(lens), n_tok=n, n_head=Hq, n_head_kv=H, d_k=dk, d_v=dv, scale=scale)
    what = f"prompt type={typ} lens={lens} H={H} G={G} dk={dk} dv={dv} pad={pad} shift={shift}"
    print(what, flush=True)
    assert dll.kvc_attn_prompt(ctypes.byref(a), None) == 0
    o, kept = so.read()
    assert kept, f"{what}: wrote between the rows"
    got_l = l.download(np.float32, n * Hq).reshape(n, Hq)
    q, k, v = (wide(s._view(s.host), typ) for s in (sq, sk, sv))
    parts = []
    with np.errstate(invalid="ignore"):
        for i, m in enumerate(lens):
            x = slice(cu[i], cu[i + 1])
            parts.append(attend(q[x], k[x], v[x], np.tril(np.ones((m, m), bool)), None, scale or 1 / np.sqrt(dk), typ))
    want = join(parts, n, Hq, dv, cu)
    inside = slice(first, first + sum(lens))
    for x in (o, got_l):
        outside = np.concatenate([x[:first], x[first + sum(lens):]])
        fill = typed(np.full(1, 7.0), typ)[0] if x is o else 9.0
        assert (outside == fill).all(), f"{what}: wrote tokens of no sequence"
    if not lse:
        assert (got_l == 9.0).all()
        got_l = want[1].astype(np.float32)
    compare(o[inside], got_l[inside].astype(np.float64), tuple(w[inside] for w in want), typ, what)
    return o[inside]


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("H,G", [(2, 1), (1, 4), (2, 3)])
def test_prompt(dll, typ, d, H, G):
    run_prompt(dll, typ, [1, 0, 37, 64, 129], H, G, d, d, seed=d + G)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
def test_prompt_longer(dll, typ):
    run_prompt(dll, typ, [300, 517, 2], 2, 2, 128, 128, seed=3, tail=5, first=3)


@pytest.mark.parametrize("typ", [F16, BF16])
@pytest.mark.parametrize("G", [1, 8])
def test_prompt_tile_edges(dll, typ, G):
    # lengths around the sizes of row and key tiles
    run_prompt(dll, typ, [15, 16, 17, 31, 33, 63, 65, 127, 128, 129, 255, 257], 1, G, 64, 64, seed=G)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("dk,dv", [(1, 1), (7, 9), (40, 24), (24, 200), (256, 3), (72, 136)])
def test_prompt_odd_heads(dll, typ, dk, dv):
    run_prompt(dll, typ, [50, 3, 41], 2, 2, dk, dv, seed=dk)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("pad,shift", [(8, 8), (1, 0), (0, 1), (4, 4)])
def test_prompt_strides(dll, typ, pad, shift):
    run_prompt(dll, typ, [70, 33], 2, 2, 64, 128, seed=pad, pad=pad, shift=shift, lse=pad != 8, scale=0.3)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("d", [64, 128, 256, 30])
def test_prompt_values_that_are_not_finite(dll, typ, d):
    # NaN and infinities of later tokens, and of the next sequence, do not reach the rows before them
    def edit(q, k, v):
        v[40, :, 5] = np.inf
        v[41, :, 5] = np.nan
        v[42, 0, 6] = -np.inf
        k[43] = np.nan
        k[60, 0, 0] = np.inf
        v[70:80] = np.nan
    run_prompt(dll, typ, [70, 10, 33], 1, 2, d, d, seed=d, edit=edit)


# ------------------------------------------------------------------ cells

def tree_masks(rng, n, words, empty=False):
    """A random tree's masks [n][words] and seen [n][n]; `empty`: one token sees not even itself."""
    seen = np.zeros((n, n), bool)
    for i in range(n):
        p = rng.integers(-1, i) if i else -1
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = True
    if empty:
        seen[n // 2] = False
    bits = np.zeros((n, words), np.uint64)
    for i in range(n):
        for j in np.nonzero(seen[i])[0]:
            if j < 64 * words:
                bits[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    seen[:, 64 * words:] = False
    return bits, seen


def run_cells(dll, typ, cache, lens, news, H, G, dk, dv, page=16, bias=False, tree=False, words=1, seed=0, pad=0,
              shift=0, max_new=None, max_len=None, layer=1, edit=None, bad_pages=(), seqs=None, empty=False, scale=0.0,
              runs=1, tail=0):
    rng = np.random.default_rng(seed)
    n_seq, Hq = len(lens), H * G
    max_pages = max(1, max(-(-m // page) for m in lens)) + 1
    n_pages = sum(-(-m // page) for m in lens) + 2
    m = PagedModel(layer + 1, n_pages, page, n_seq + 2, max_pages, H, dk, dv, cache, cache, bias)
    order, at = rng.permutation(n_pages), 0
    place = rng.permutation(n_seq + 2)[:n_seq] if seqs is None else np.asarray(seqs)
    for s, n in zip(place, lens):
        if not 0 <= s < n_seq + 2:
            continue
        p = -(-n // page)
        m.table[s, :p] = order[at:at + p]
        m.len[s] = n
        at += p
    k = rng.standard_normal((n_pages, page, H, dk)) * np.exp(0.5 * rng.standard_normal((H, dk)))
    v = rng.standard_normal((n_pages, page, H, dv))
    n = sum(news) + tail
    q = rng.standard_normal((n, Hq, dk)) + 0.4 * k[0, 0].repeat(G, 0)
    if bias:
        m.bias[:] = rng.standard_normal(m.bias.shape) * 2
    cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)

    def cell(s, j):
        """(page, cell) of cell j of the call's sequence s"""
        return m.table[place[s], j // page], j % page

    if edit:
        edit(q, k, v, m.bias[layer] if bias else None, cell)
    with np.errstate(over="ignore", invalid="ignore"):
        m.K[layer] = encode(k.reshape(n_pages, page, -1), cache)
        m.V[layer] = encode(v.reshape(n_pages, page, -1), cache)
    # what no sequence holds is garbage
    used = np.zeros((n_pages, page), bool)
    for s in range(n_seq):
        if 0 <= place[s] < n_seq + 2:
            for j in range(lens[s]):
                used[cell(s, j)] = True
    m.K[layer][~used] = 0xFF
    m.V[layer][~used] = 0xFF
    if bias:
        m.bias[layer].transpose(0, 2, 1)[~used] = np.nan
    K, V = (decode(x[layer], cache).reshape(n_pages, page, H, -1) for x in (m.K, m.V))
    parts, masks = [], []
    sq = Strided(q, typ, pad, shift)
    qd = wide(sq._view(sq.host), typ)
    for s in range(n_seq):
        nn, L = news[s], lens[s]
        good = 0 <= place[s] < n_seq + 2 and nn <= L
        bits, see = tree_masks(rng, nn, words, empty) if tree else (np.zeros((nn, 1), np.uint64), np.tril(np.ones((nn, nn), bool)))
        masks.append(bits)
        if not good:
            parts.append((np.zeros((nn, Hq, dv)), np.full((nn, Hq), -np.inf), np.full((nn, Hq, dv), 1e-30), np.zeros((nn, Hq))))
            continue
        seen = np.ones((nn, L), bool)
        seen[:, L - nn:] = see
        row = m.table[place[s]].copy()
        for (b, col, value) in bad_pages:
            if b == s:
                seen[:, col * page:(col + 1) * page] = False
        p, c = m.spots(row, np.arange(L))
        b = m.bias[layer][p, :, c].T.astype(np.float64) if bias else None
        with np.errstate(invalid="ignore"):
            parts.append(attend(qd[cu[s]:cu[s + 1]], K[p, c], V[p, c], seen, b, scale or 1 / np.sqrt(dk), typ))
    for (b, col, value) in bad_pages:
        m.table[place[b], col] = value
    want = join(parts, n, Hq, dv, cu)
    bufs = {x: dev(getattr(m, x)) for x in ("K", "V", "table", "len", "refs")}
    db = dev(m.bias) if bias else None
    c = kc.KvCache(n_layers=layer + 1, n_pages=n_pages, page_size=page, max_seqs=n_seq + 2, max_pages=max_pages,
                   n_head_kv=H, d_k=dk, d_v=dv, k_type=cache, v_type=cache, bias=db.value if bias else None,
                   **{x: y.value for x, y in bufs.items()})
    so = Strided(np.full((n, Hq, dv), 7.0), typ, pad, shift)
    lse = dev(np.full((n, Hq), 9.0, np.float32))
    extra = [dev(np.int32(place)), dev(cu), dev(np.concatenate(masks) if masks else np.zeros(1, np.uint64))]
    a = kc.CacheAttnArgs(q=sq.heads(), o=so.heads(), lse=lse.value, seqs=extra[0].value, cu=extra[1].value,
                         mask=extra[2].value if tree else None, mask_words=words if tree else 0, layer=layer, type=typ,
                         n_seq=n_seq, n_tok=n, n_head=Hq, max_new=max(news) if max_new is None else max_new,
                         max_len=max(lens) if max_len is None else max_len, scale=scale)
    size = dll.kvc_attn_cache_workspace(ctypes.byref(c), ctypes.byref(a))
    ws = dev(np.full(max(size, 16), 0xFF, np.uint8))
    what = (f"cells type={typ} cache={cache} lens={lens} news={news} H={H} G={G} dk={dk} dv={dv} page={page} bias={bias} "
            f"tree={tree} ws={size}")
    print(what, flush=True)
    first = None
    for _ in range(runs):
        assert dll.kvc_attn_cache(ctypes.byref(c), ctypes.byref(a), ws.value, size, None) == 0
        o, kept = so.read()
        assert kept, f"{what}: wrote between the rows"
        l = lse.download(np.float32, n * Hq).reshape(n, Hq)
        e = sum(news)
        assert (o[e:] == typed(np.full(1, 7.0), typ)[0]).all() and (l[e:] == 9.0).all(), f"{what}: wrote past the last sequence"
        compare(o[:e], l[:e].astype(np.float64), tuple(w[:e] for w in want), typ, what)
        if first is None:
            first = o.copy()
        assert np.array_equal(first.view(np.uint8), o.view(np.uint8)), f"{what}: two runs differ"
    if size:
        assert dll.kvc_attn_cache(ctypes.byref(c), ctypes.byref(a), ws.value, size - 1, None) == kc.E_SCRATCH
        assert dll.kvc_attn_cache(ctypes.byref(c), ctypes.byref(a), None, size, None) == -1
    return o


KINDS = [(F16, F16), (BF16, BF16), (F32, F32), (F16, Q8_0), (BF16, Q8_0)]


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("bias", [False, True])
def test_single_tokens(dll, typ, cache, d, bias):
    run_cells(dll, typ, cache, [1, 2, 33, 170, 64], [1, 1, 1, 1, 1], 2, 4, d, d, bias=bias, seed=d, tail=2)


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 128])
def test_trees(dll, typ, cache, d, page):
    run_cells(dll, typ, cache, [300, 13, 64, 130], [13, 13, 5, 40], 2, 2, d, d, page=page, bias=page == 16, tree=True,
              seed=d + page)


@pytest.mark.parametrize("typ,cache", KINDS)
def test_causal_chunks(dll, typ, cache):
    # no mask: each new token sees the cells up to its own
    run_cells(dll, typ, cache, [200, 50, 31], [77, 50, 1], 1, 3, 128, 128, page=32, seed=4)


@pytest.mark.parametrize("typ,cache", KINDS)
def test_key_ranges(dll, typ, cache):
    # long enough to be cut into ranges that are joined afterwards; some ranges of the shorter sequences are empty
    run_cells(dll, typ, cache, [2300, 1, 700], [1, 1, 1], 1, 5, 128, 64 if cache != Q8_0 else 128, page=64, bias=True,
              seed=5, runs=2)
    run_cells(dll, typ, cache, [1900, 90], [20, 9], 2, 1, 64, 64, page=16, tree=True, seed=6, runs=2)


@pytest.mark.parametrize("typ,cache", KINDS)
def test_larger_than_said(dll, typ, cache):
    # max_new and max_len shape the launch: more tokens and cells than they say are computed all the same
    run_cells(dll, typ, cache, [900, 120], [70, 3], 1, 2, 64, 64, tree=True, words=2, seed=7, max_new=1, max_len=1)


@pytest.mark.parametrize("words", [1, 2, 3])
def test_mask_words(dll, words):
    run_cells(dll, BF16, BF16, [260, 150], [140, 65], 1, 2, 64, 64, tree=True, words=words, seed=words)


@pytest.mark.parametrize("typ,cache", KINDS)
def test_rows_that_see_nothing(dll, typ, cache):
    # no committed cells, and a token whose mask is empty; more tokens than cells; a bad sequence number
    run_cells(dll, typ, cache, [6, 4, 40, 9], [6, 5, 2, 3], 1, 2, 64, 64, tree=True, seed=8, empty=True,
              seqs=[0, 3, -1, 77])


@pytest.mark.parametrize("typ,cache", KINDS)
def test_bias_that_hides(dll, typ, cache):
    # -inf hides a cell for its head, whatever its rows hold; the lowest value does not when a row has nothing else
    low = np.finfo(np.float32).min

    def edit(q, k, v, b, cell):
        for j in range(20, 40):
            p, c = cell(0, j)
            b[p, :, c] = -np.inf
            k[p, c] = np.nan if cache != Q8_0 else 1.0
            v[p, c, :, ::3] = np.inf if cache != Q8_0 else 1.0
        for j in range(50):
            p, c = cell(1, j)
            b[p, 0, c] = -np.inf        # nothing left for head 0
            b[p, 1, c] = low            # nothing but the lowest for head 1
    run_cells(dll, typ, cache, [90, 50], [2, 1], 2, 2, 64, 64, bias=True, seed=9, edit=edit)


@pytest.mark.parametrize("typ,cache", [k for k in KINDS if k[1] != Q8_0])
@pytest.mark.parametrize("d", [64, 128, 256, 20])
def test_drafts_that_are_not_finite(dll, typ, cache, d):
    # what a drafted token holds reaches only the tokens that see it
    def edit(q, k, v, b, cell):
        for j, x in ((91, np.inf), (93, np.nan), (95, -np.inf)):
            p, c = cell(0, j)
            v[p, c, :, 3::5] = x
        p, c = cell(0, 97)
        k[p, c] = np.nan
        q[3, 0, 0] = np.nan
    run_cells(dll, typ, cache, [100], [12], 1, 2, d, d, tree=True, seed=d, edit=edit)


@pytest.mark.parametrize("typ,cache", KINDS)
def test_bad_pages_are_not_seen(dll, typ, cache):
    run_cells(dll, typ, cache, [150, 80, 20], [3, 1, 2], 1, 2, 64, 64, page=16, seed=10, bias=True,
              bad_pages=[(0, 1, 1 << 20), (0, 4, -1), (1, 0, -7), (2, 0, 1 << 30)])


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("dk,dv,pad,shift", [(7, 9, 0, 0), (64, 64, 1, 0), (128, 64, 0, 1), (33, 250, 0, 0), (64, 128, 8, 8)])
def test_odd_heads_and_strides(dll, typ, dk, dv, pad, shift):
    run_cells(dll, typ, typ, [100, 45], [7, 1], 2, 2, dk, dv, page=16, bias=True, tree=True, seed=dk, pad=pad,
              shift=shift, scale=0.2)


@pytest.mark.parametrize("typ,cache", [(F32, F32), (F16, Q8_0), (BF16, Q8_0)])
def test_wide_ranges_of_values(dll, typ, cache):
    # scales of the rows from 2^-10 to 2^10: no form may depend on values near one
    def edit(q, k, v, b, cell):
        v *= np.exp2(np.random.default_rng(1).integers(-10, 11, v.shape[:3]))[..., None]
        k *= np.exp2(np.random.default_rng(2).integers(-10, 3, k.shape[:3]))[..., None]
    run_cells(dll, typ, cache, [200], [3], 2, 2, 128, 128, page=32, seed=11, edit=edit)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("d", [64, 256])
def test_negative_scale(dll, typ, d):
    # the largest score is then that of the smallest product
    run_prompt(dll, typ, [5, 140], 1, 2, d, d, seed=20, scale=-0.1)
    run_cells(dll, typ, typ, [150, 30], [3, 1], 1, 2, d, d, tree=True, bias=True, seed=21, scale=-0.1)
    run_cells(dll, typ, typ, [190, 80], [70, 40], 1, 2, d, d, tree=True, words=2, seed=22, scale=-0.1)


@pytest.mark.parametrize("typ", [F16, BF16])
def test_many_prompts(dll, typ):
    # more sequences than a wave has lanes, empty ones among them
    run_prompt(dll, typ, [(7 * i) % 5 * 9 for i in range(150)], 1, 2, 64, 64, seed=23, first=2, tail=3)


@pytest.mark.parametrize("typ,cache", [(F16, F16), (BF16, Q8_0)])
def test_many_sequences(dll, typ, cache):
    run_cells(dll, typ, cache, [1 + 11 * i % 60 for i in range(150)], [1 + i % 2 if 1 + 11 * i % 60 > 1 else 1 for i in range(150)],
              1, 2, 64, 64, seed=24, bias=True)


@pytest.mark.parametrize("typ", [F16, BF16])
@pytest.mark.parametrize("d,said", [(64, 17), (64, 40), (96, 17), (96, 40), (128, 40), (256, 17), (256, 40), (200, 40)])
def test_trees_of_several_row_tiles(dll, typ, d, said):
    # a block that takes several tiles of rows, one after the other, where more tokens come than were announced; heads
    # narrower than the form; what the next row tile finds in LDS
    run_cells(dll, typ, typ, [700, 290, 200], [140, 129, 3], 2, 2, d, d, page=32, bias=d != 96, tree=True, words=3, seed=d + said,
              max_new=said, max_len=200, runs=2)


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("G", [7, 40, 100])
def test_large_groups(dll, typ, cache, G):
    run_cells(dll, typ, cache, [300, 20, 5], [1, 2, 3], 1, G, 64, 64, tree=True, seed=G)


@pytest.mark.parametrize("typ", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,G", [(12, 1), (12, 2), (10, 4), (20, 4)])
def test_q8_rows_that_are_not_finite(dll, typ, d, n, G):
    # scales of drafted tokens that are not finite, or far from one, with few and many rows
    def edit(q, k, v, b, cell):
        for j, x in ((101, 1e-7), (102, 2e3), (103, 2.0 ** -20), (105, 1e8)):
            p, c = cell(0, j)
            v[p, c, 0, :32] *= x
    run_cells(dll, typ, Q8_0, [100 + n], [n], 1, G, d, d, tree=True, bias=True, seed=d + n, edit=edit)


@pytest.mark.parametrize("typ", [F16, BF16])
@pytest.mark.parametrize("G", [1, 3, 12])
def test_q8_queries_of_any_alignment(dll, typ, G):
    run_cells(dll, typ, Q8_0, [100, 45], [7, 1], 2, G, 96, 64, bias=True, tree=True, seed=25, pad=1, shift=1)
    run_cells(dll, typ, Q8_0, [100, 45], [7, 1], 1, G, 128, 128, seed=26, pad=3, shift=1)


@pytest.mark.parametrize("typ,cache", KINDS)
def test_nothing_announced(dll, typ, cache):
    # max_new and max_len 0; a sequence without cells beside others; one without tokens
    run_cells(dll, typ, cache, [40, 0, 9], [40, 0, 0], 2, 2, 64, 64, seed=27, max_new=0, max_len=0)


@pytest.mark.parametrize("typ,cache", KINDS)
def test_the_same_sequence_twice(dll, typ, cache):
    # (reads only: each entry sees the whole sequence)
    run_cells(dll, typ, cache, [90, 90, 50], [3, 3, 3], 1, 2, 64, 64, seed=28, seqs=[2, 2, 0])


@pytest.mark.parametrize("typ", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128, 136, 200, 256])
@pytest.mark.parametrize("G", [1, 3])
def test_longer_prompts(dll, typ, d, G):
    # tiles that every row sees whole, then those with hidden keys; values that are not finite in both
    def edit(q, k, v):
        v[9, :, 5] = np.inf
        v[260, 0, d - 1] = -np.inf
        v[290, :, 7] = np.nan
        v[400:, :, 3] = np.inf
        k[299] = np.nan
    run_prompt(dll, typ, [300, 333, 66], 2, G, d, d, seed=30 + d, edit=edit)
    run_prompt(dll, typ, [300, 333, 66], 1, G, d, d, seed=31 + d, tail=2)
