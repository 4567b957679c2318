"""Pages of the paged cache (include/kvc-cache.h) against a model on the host:
every array, rows and free pages' old contents among them, after each call."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from cache_model import BAD, BF16, F16, F32, PagedModel, Q8_0, encode
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


class Cache:
    """A cache on the device beside its model."""

    def __init__(self, dll, seed=0, L=2, pages=24, page=16, seqs=6, max_pages=12, H=2, dk=32, dv=32, k_type=F16,
                 v_type=F16, bias=True):
        self.dll, self.rng = dll, np.random.default_rng(seed)
        m = self.m = PagedModel(L, pages, page, seqs, max_pages, H, dk, dv, k_type, v_type, bias)
        m.K[:] = self.rng.integers(0, 256, m.K.shape, np.uint8)
        m.V[:] = self.rng.integers(0, 256, m.V.shape, np.uint8)
        if bias:
            m.bias[:] = self.rng.standard_normal(m.bias.shape, np.float32)
        self.bufs = {n: dev(getattr(m, n)) for n in ("K", "V", "table", "len", "refs")}
        self.bufs["bias"] = dev(m.bias) if bias else None
        self.c = kc.KvCache(n_layers=L, n_pages=pages, page_size=page, max_seqs=seqs, max_pages=max_pages, n_head_kv=H,
                            d_k=dk, d_v=dv, k_type=k_type, v_type=v_type,
                            **{n: b.value if b else None for n, b in self.bufs.items()})
        self.keep = []

    def ws(self, n):
        size = self.dll.kvc_cache_workspace(ctypes.byref(self.c), n)
        assert size
        self.keep = [dev(np.full(size, 0xA5, np.uint8))]
        return self.keep[0].value, size

    def check(self, what):
        m = self.m
        for n in ("table", "len", "refs", "K", "V", "bias"):
            a = getattr(m, n)
            if a is None:
                continue
            b = self.bufs[n].download(a.dtype, a.size).reshape(a.shape)
            if a.dtype == np.float32:
                a, b = a.view(np.uint32), b.view(np.uint32)
            assert np.array_equal(a, b), f"{what}: {n} differs at {np.argwhere(a != b)[:4].tolist()}"
        # counts are those of the tables
        assert np.array_equal(m.refs, np.bincount(m.table[m.table >= 0], minlength=m.n_pages)), what

    def _status(self, rc, want, buf, what):
        assert rc == 0, f"{what}: {rc}"
        got = buf.download(np.int32, len(want)).tolist()
        assert got == want, f"{what}: status {got}, expected {want}"
        self.check(what)

    def extend(self, seqs, counts):
        st = dev(np.full(len(seqs), 77, np.int32))
        a, b = dev(np.int32(seqs)), dev(np.int32(counts))
        rc = self.dll.kvc_cache_extend(self.c, len(seqs), a.value, b.value, st.value, *self.ws(len(seqs)), None)
        self._status(rc, self.m.extend(seqs, counts), st, f"extend {seqs} {counts}")

    def write(self, seqs, counts, layer=0, n_layers=None, src_type=None, pad=0):
        m = self.m
        n_layers = m.L - layer if n_layers is None else n_layers
        cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        n = int(cu[-1])
        src_type = m.k_type if src_type is None else src_type
        rows, bufs = [], []
        for d in (m.dk, m.dv):
            x = self.rng.standard_normal((n_layers, n, m.H * d)).astype(np.float32)
            x = x * np.exp(self.rng.standard_normal((n_layers, n, 1))).astype(np.float32)
            if src_type == BF16:
                x = (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
            elif src_type == F16:
                x = x.astype(np.float16).astype(np.float32)
            b = encode(x, src_type)
            wide = np.zeros((n_layers, n, b.shape[2] + pad), np.uint8)
            wide[..., :b.shape[2]] = b
            buf = dev(wide)
            bufs.append(buf)
            rows.append((encode(x, m.k_type), kc.Rows(buf.value, n * wide.shape[2], wide.shape[2])))
        a, b = dev(np.int32(seqs)), dev(cu)
        rc = self.dll.kvc_cache_write(self.c, layer, n_layers, len(seqs), a.value, b.value, n, src_type,
                                      ctypes.byref(rows[0][1]), ctypes.byref(rows[1][1]), None)
        assert rc == 0
        m.write(layer, n_layers, seqs, cu, rows[0][0], rows[1][0])
        self.check(f"write {seqs} {counts}")

    def fork(self, src, dst):
        st = dev(np.full(len(src), 77, np.int32))
        a, b = dev(np.int32(src)), dev(np.int32(dst))
        rc = self.dll.kvc_cache_fork(self.c, len(src), a.value, b.value, st.value, None)
        self._status(rc, self.m.fork(src, dst), st, f"fork {src} {dst}")

    def free(self, seqs):
        a = dev(np.int32(seqs))
        assert self.dll.kvc_cache_free(self.c, len(seqs), a.value, None) == 0
        self.m.free(seqs)
        self.check(f"free {seqs}")

    def compact(self, seqs, start, kept, same=False, values=False, betas=False, heads_apart=False):
        """kept: per sequence, per layer (or one list for all) the ascending indices from start."""
        m = self.m
        n = [len(k[0]) for k in kept]
        cu = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        total = int(cu[-1])
        idx = np.zeros((1 if same else m.L, max(total, 1)), np.int32)
        for i, k in enumerate(kept):
            for l in range(idx.shape[0]):
                idx[l, cu[i]:cu[i + 1]] = k[l]
        full = np.repeat(idx, m.L, 0) if same else idx
        v = beta = pv = pb = None
        bufs = [dev(np.int32(seqs)), dev(np.int32(start)), dev(cu), dev(idx), dev(np.full(len(seqs), 77, np.int32))]
        if values:
            v = self.rng.integers(0, 256, (m.L, total, m.V.shape[3]), np.uint8)
            hb = v.shape[2] // m.H
            if heads_apart:   # [L][H][rows][head bytes], as refitted values stand
                bufs.append(dev(v.reshape(m.L, total, m.H, hb).transpose(0, 2, 1, 3)))
                pv = kc.Values(bufs[-1].value, m.H * total * hb, hb, total * hb)
            else:
                bufs.append(dev(v))
                pv = kc.Values(bufs[-1].value, total * m.H * hb, m.H * hb, hb)
        if betas:
            beta = self.rng.standard_normal((m.L, m.H, total), np.float32)
            bufs.append(dev(beta))
            pb = kc.Betas(bufs[-1].value, m.H * total, total)
        rc = self.dll.kvc_cache_compact(self.c, len(seqs), bufs[0].value, bufs[1].value, bufs[2].value, total,
                                        bufs[3].value, 0 if same else idx.shape[1], ctypes.byref(pv) if pv else None,
                                        ctypes.byref(pb) if pb else None, bufs[4].value, *self.ws(len(seqs)), None)
        want = m.compact(seqs, start, cu, full, v, beta)
        self._status(rc, want, bufs[4], f"compact {seqs} from {start} keeping {n}")

    def some(self, n, k):
        return np.sort(self.rng.choice(n, k, replace=False)).astype(np.int32)


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("kt,vt,dk,dv,H", [(F16, F16, 32, 32, 2), (F32, F32, 5, 3, 1), (BF16, BF16, 9, 8, 3),
                                           (Q8_0, Q8_0, 32, 64, 2), (F16, F32, 128, 128, 8)])
def test_a_sequence_of_calls(dll, page, kt, vt, dk, dv, H):
    c = Cache(dll, seed=page + kt, page=page, H=H, dk=dk, dv=dv, k_type=kt, v_type=vt)
    same = kt == vt
    c.extend([0, 1, 2], [2 * page + 3, page, 0])
    if same:
        c.write([0, 1, 2], [2 * page + 3, page, 0], pad=0 if kt == F32 else 2)
    c.fork([0, 1, 2], [3, 4, 5])
    # shared partly filled pages are copied, whole ones are not
    c.extend([3, 4, 0], [1, 1, 0])
    if same:
        c.write([3, 4], [1, 1], layer=1, n_layers=1)
    c.extend([0, 3], [page, 2 * page])
    c.free([1, 1, 5, 77, -1])
    # drafts accepted: the tail moves up inside its own pages
    n = int(c.m.len[3])
    c.compact([3], [n - 5], [[[0, 2, 4]]], same=True)
    # cut to a length, inside a page and at its edge
    c.compact([3, 4], [page + 2, page], [[[]], [[]]], same=True)
    # in place over the whole length, another set in each layer
    n = int(c.m.len[0])
    c.compact([0], [0], [[c.some(n, n // 2), c.some(n, n // 2)]])
    c.free([0, 1, 2, 3, 4, 5])
    assert not c.m.refs.any()


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("heads_apart", [False, True])
def test_compaction_of_shared_pages(dll, bias, heads_apart):
    c = Cache(dll, seed=5, pages=40, page=16, max_pages=30, bias=bias, L=3)
    c.extend([0], [200])
    c.write([0], [200])
    c.fork([0, 0], [1, 2])
    # every page has other holders: fresh pages, from the first cell on
    c.compact([1], [0], [[c.some(200, 77) for _ in range(3)]], values=True, betas=bias, heads_apart=heads_apart)
    # from the middle of a shared page: its leading cells come along
    c.compact([2], [37], [[c.some(163, 20) for _ in range(3)]], values=heads_apart)
    # the original is its own again on most pages
    c.compact([0], [3], [[c.some(197, 150) for _ in range(3)]], betas=bias)
    # two of one set of pages at once
    c.free([1, 2])
    c.fork([0], [1])
    c.compact([0, 1], [0, 20], [[c.some(153, 40) for _ in range(3)], [c.some(133, 30) for _ in range(3)]])


def test_long_compaction_in_place(dll):
    # more cells than a block works out at a time, an in-place chain through every page
    c = Cache(dll, seed=9, L=2, pages=300, page=16, seqs=2, max_pages=300, H=1, dk=16, dv=48)
    c.extend([0], [4000])
    c.write([0], [4000])
    c.compact([0], [1], [[c.some(3999, 3500), c.some(3999, 3500)]])
    c.compact([0], [0], [[np.arange(3501)]], same=True)          # nothing moves
    c.compact([0], [0], [[np.arange(1, 3501)]], same=True)       # every cell by one


def test_pages_that_are_missing(dll):
    c = Cache(dll, pages=6, page=16, max_pages=8)
    c.extend([0], [40])                      # 3 pages
    c.extend([1, 2, 3], [64, 17, 1])         # 4 pages are not there, 2 are, none is left
    c.fork([0], [4])
    c.extend([4], [1])                       # the copy of the shared page is not there
    c.free([2])
    c.extend([4], [1])
    c.extend([4, 4, 1], [8, 8, 1])           # named twice
    c.compact([0, 4], [0, 0], [[[1, 5]], [[0, 9]]], same=True)   # both share their first page, one page is free
    c.extend([9, 0, 1, 5], [1, -1, 200, 0])  # bad number, bad count, more than a table holds, nothing


def test_many_requests(dll):
    c = Cache(dll, pages=3000, page=16, seqs=1024, max_pages=4, L=1, H=1)
    seqs = np.random.default_rng(1).permutation(1024)
    counts = np.random.default_rng(2).integers(0, 40, 1024)
    c.extend(seqs.tolist(), counts.tolist())
    c.free(seqs[:500].tolist())
    c.fork(seqs[500:1000].tolist(), seqs[:500].tolist())
    c.extend(seqs.tolist(), np.random.default_rng(3).integers(0, 9, 1024).tolist())


@pytest.mark.parametrize("src", [F32, F16, BF16])
def test_rows_encoded_into_q8_0(dll, src):
    c = Cache(dll, k_type=Q8_0, v_type=Q8_0, dk=64, dv=32, H=3)
    c.extend([1, 0], [21, 3])
    c.write([1, 0], [21, 3], src_type=src)


def test_write_of_rows_that_have_no_cell(dll):
    # more rows than the sequence has cells, a bad sequence, and an empty one
    c = Cache(dll)
    c.extend([0], [4])
    c.write([0, 40, 1], [6, 2, 1])


def test_read(dll):
    c = Cache(dll, page=16, dk=48, dv=7, L=3)
    c.extend([0, 2], [50, 33])
    c.write([0, 2], [50, 33])
    m = c.m
    for start, count in [(0, 33), (5, 40), (30, 9), (100, 2), (0, 1)]:
        K, V, B = (np.full(s, 0x77, np.uint8) for s in ((m.L, count, m.K.shape[3]), (m.L, count, m.V.shape[3]),
                                                        (m.L, m.H, count, 4)))
        dk, dv, db = dev(K), dev(V), dev(B)
        assert c.dll.kvc_cache_read(c.c, 2, start, count, dk.value, dv.value, db.value, None) == 0
        n = max(0, min(count, 33 - start))
        p, e = m.spots(m.table[2], np.arange(start, start + n))
        for pool, buf in ((m.K, dk), (m.V, dv)):
            want = np.zeros((m.L, count, pool.shape[3]), np.uint8)
            want[:, :n] = pool[:, p, e]
            assert np.array_equal(buf.download(np.uint8, want.size).reshape(want.shape), want), (start, count)
        want = np.zeros((m.L, m.H, count), np.float32)
        want[..., :n] = m.bias[:, p, :, e].transpose(1, 2, 0)
        assert np.array_equal(db.download(np.float32, want.size).reshape(want.shape), want)


def test_reset(dll):
    c = Cache(dll)
    c.extend([0, 1], [20, 20])
    assert c.dll.kvc_cache_reset(c.c, None) == 0
    c.m.table[:], c.m.len[:], c.m.refs[:] = -1, 0, 0
    c.check("reset")


def test_bad_state_is_left_alone(dll):
    # a table that names pages the cache does not have: requests on it are refused, and nothing is read or written there
    c = Cache(dll)
    c.extend([0, 1], [20, 20])
    import hiprt
    t = c.m.table.copy()
    t[0, 1] = 1 << 24
    t[1, 1] = -5
    c.bufs["table"].upload(t)
    st = dev(np.full(2, 77, np.int32))
    a, k, z = dev(np.int32([0, 1])), dev(np.int32([1, 1])), dev(np.int32([0, 0, 0]))
    assert c.dll.kvc_cache_extend(c.c, 2, a.value, k.value, st.value, *c.ws(2), None) == 0
    assert st.download(np.int32, 2).tolist() == [BAD, BAD]
    assert c.dll.kvc_cache_compact(c.c, 2, a.value, z.value, z.value, 0, None, 0, None, None, st.value, *c.ws(2), None) == 0
    assert st.download(np.int32, 2).tolist() == [BAD, BAD]
    hiprt.synchronize()
    c.bufs["table"].upload(c.m.table)
    c.check("after refusals")
