"""Steps that the cache refuses in part (include/kvc-cache.h): reservations that
find no page and the writes and attention queued behind them, and compactions
whose indices do not fit. What nobody asked to change is as it was."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from cache_model import BAD, BF16, F16, F32, Q8_0, attend, decode, encode
from kvc_harness import kc
from test_gpu_cache_attn import Strided, compare, wide
from test_gpu_cache_pages import Cache, dev, dll   # noqa: F401 (the fixture)
from test_gpu_cache_run import _graph_api

pytestmark = pytest.mark.gpu


def test_a_shared_page_is_not_written(dll):   # noqa: F811
    c = Cache(dll, pages=4, page=16, max_pages=8, L=2)
    c.extend([0], [24])
    c.write([0], [24])
    c.fork([0], [1])
    c.extend([2], [32])                      # the two pages that were free
    c.write([2], [32])
    c.extend([1], [1])                       # the copy of the shared page is not there
    assert c.m.len[1] == 24
    rows, cu, seqs = dev(np.full(2 * 128, 0x11, np.uint8)), dev(np.int32([0, 1])), dev(np.int32([1]))
    r = kc.Rows(rows.value, 128, 128)
    assert dll.kvc_cache_write(c.c, 0, 2, 1, seqs.value, cu.value, 1, F16, r, r, None) == 0
    c.check("a write behind a refused extend, into a shared page")
    # a row for each sequence and a longer one: only pages that are a sequence's own take theirs
    rows, cu, seqs = dev(np.full(11 * 128, 0x22, np.uint8)), dev(np.int32([0, 1, 10, 11])), dev(np.int32([0, 2, 1]))
    r = kc.Rows(rows.value, 0, 128)
    assert dll.kvc_cache_write(c.c, 1, 1, 3, seqs.value, cu.value, 11, F16, r, r, None) == 0
    x = np.full((1, 11, 128), 0x22, np.uint8)
    c.m.write(1, 1, [2], [1, 10], x, x)
    c.check("own pages beside shared ones")


def test_sequences_that_were_granted(dll):   # noqa: F811
    c = Cache(dll, pages=6, page=16, max_pages=4, seqs=6, L=1)
    c.extend([0, 1, 4], [20, 32, 5])
    c.write([0, 1, 4], [20, 32, 5])
    # done; done without a page; a bad count; named twice; no such sequence; a page that is missing; nothing asked
    seqs, counts = [1, 0, 4, 1, 77, 2, 5, -3], [1, 3, -1, 1, 1, 33, 0, 1]
    want = c.m.extend(seqs, counts)
    assert want == [0, 0, BAD, BAD, BAD, 3, 0, BAD]
    a, k, st, g = dev(np.int32(seqs)), dev(np.int32(counts)), dev(np.full(8, 77, np.int32)), dev(np.full(9, 55, np.int32))
    assert dll.kvc_cache_extend_granted(c.c, 8, a.value, k.value, st.value, g.value, *c.ws(8), None) == 0
    c._status(0, want, st, "extend, granted")
    assert g.download(np.int32, 9).tolist() == [1, 0, -1, -1, -1, -1, 5, -1, 55]
    # the numbers in place of the ones asked for
    want = c.m.extend(seqs, counts)
    assert dll.kvc_cache_extend_granted(c.c, 8, a.value, k.value, st.value, a.value, *c.ws(8), None) == 0
    c._status(0, want, st, "extend, granted in place")
    assert a.download(np.int32, 8).tolist() == [s if w == 0 else -1 for s, w in zip(seqs, want)]


def test_a_step_behind_a_refused_reservation(dll):   # noqa: F811
    """Reserve, write and attend queued together, eager and as a graph that is replayed while the pool runs out: refused
    sequences keep their cells, and their tokens see nothing."""
    import hiprt
    h = _graph_api()
    H, G, d, page = 2, 2, 32, 16
    c = Cache(dll, pages=5, page=page, max_pages=4, seqs=4, L=1, H=H, dk=d, dv=d)
    c.extend([0, 1, 2], [14, 32, 15])        # one page is left
    c.write([0, 1, 2], [14, 32, 15])
    c.m.bias[:, c.m.table[2, 0], :, :] = -np.inf   # (nothing of sequence 2 is to be seen, committed or not)
    c.bufs["bias"].upload(c.m.bias)
    seqs, counts = [1, 0, 2], [1, 1, 1]
    a, k, cu = dev(np.int32(seqs)), dev(np.int32(counts)), dev(np.int32([0, 1, 2, 3]))
    st, granted = dev(np.zeros(3, np.int32)), dev(np.zeros(3, np.int32))
    rng = np.random.default_rng(8)
    rows = [dev(np.zeros(3 * H * d * 2, np.uint8)) for _ in range(2)]
    r = [kc.Rows(x.value, 0, 2 * H * d) for x in rows]
    q, o = Strided(rng.standard_normal((3, H * G, d)), F16), Strided(np.full((3, H * G, d), 7.0), F16)
    lse = dev(np.full((3, H * G), 9.0, np.float32))
    x = kc.CacheAttnArgs(q=q.heads(), o=o.heads(), lse=lse.value, seqs=granted.value, cu=cu.value, type=F16, n_seq=3, n_tok=3,
                         n_head=H * G, max_new=1, max_len=64)
    ws = c.ws(3)
    assert dll.kvc_attn_cache_workspace(c.c, x) == 0

    def step(stream):
        assert dll.kvc_cache_extend_granted(c.c, 3, a.value, k.value, st.value, granted.value, *ws, stream) == 0
        assert dll.kvc_cache_write(c.c, 0, 1, 3, granted.value, cu.value, 3, F16, r[0], r[1], stream) == 0
        assert dll.kvc_attn_cache(c.c, x, None, 0, stream) == 0

    stream, graph, exe = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    hiprt.check(h.hipStreamCreate(ctypes.byref(stream)))
    hiprt.check(h.hipStreamBeginCapture(stream, 2))
    step(stream)
    hiprt.check(h.hipStreamEndCapture(stream, ctypes.byref(graph)))
    hiprt.check(h.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0))
    refused = 0
    for i in range(6):
        new = [rng.standard_normal((3, H * d)).astype(np.float16).astype(np.float32) for _ in range(2)]
        for b, y in zip(rows, new):
            b.upload(encode(y, F16))
        want = c.m.extend(seqs, counts)
        c.m.write(0, 1, [s if w == 0 else -1 for s, w in zip(seqs, want)], [0, 1, 2, 3], *(encode(y, F16)[None] for y in new))
        hiprt.synchronize()
        if i % 2:
            step(None)
        else:
            hiprt.check(h.hipGraphLaunch(exe, stream))
        hiprt.synchronize()
        c._status(0, want, st, f"step {i}")
        refused += sum(w != 0 for w in want)
        got, kept = o.read()
        assert kept
        l = lse.download(np.float32, 3 * H * G).reshape(3, H * G)
        qd = wide(q._view(q.host), F16)
        for j, (s, w) in enumerate(zip(seqs, want)):
            if w:
                assert not got[j].any() and (l[j] == -np.inf).all(), f"step {i}: tokens of a refused request"
                continue
            n = int(c.m.len[s])
            p, e = c.m.spots(c.m.table[s], np.arange(n))
            K, V = (decode(z[0][p, e], F16).reshape(n, H, d) for z in (c.m.K, c.m.V))
            ref = attend(qd[j:j + 1], K, V, np.ones((1, n), bool), c.m.bias[0][p, :, e].T.astype(float), d ** -0.5, F16)
            compare(got[j:j + 1], l[j:j + 1].astype(float), ref, F16, f"step {i}, sequence {s}")
    assert refused >= 3
    hiprt.check(h.hipGraphExecDestroy(exe))
    hiprt.check(h.hipGraphDestroy(graph))
    hiprt.check(h.hipStreamDestroy(stream))

class BadIndices(Cache):
    """Compactions some of whose indices do not fit."""

    def run(self, seqs, start, cu, idx, total, values=False, betas=False, bad=(), what=""):
        """idx [L][cu[-1]] as handed over; total the n_idx of the call; bad: (layer, k) of cells to be left unwritten."""
        m = self.m
        cu, idx = np.int32(cu), np.int32(idx)
        n = idx.shape[1]
        good = idx.copy()
        for l, k in bad:
            i = np.searchsorted(cu[1:], k, side="right")
            good[l, k] = k - cu[i]           # (what the model moves; put back below)
        bufs = [dev(np.int32(seqs)), dev(np.int32(start)), dev(cu), dev(idx), dev(np.full(len(seqs), 77, np.int32))]
        v = beta = pv = pb = None
        if values:
            v = self.rng.integers(0, 256, (m.L, n, m.V.shape[3]), np.uint8)
            bufs.append(dev(v))
            pv = kc.Values(bufs[-1].value, n * v.shape[2], v.shape[2], v.shape[2] // m.H)
        if betas:
            beta = self.rng.standard_normal((m.L, m.H, n), np.float32)
            bufs.append(dev(beta))
            pb = kc.Betas(bufs[-1].value, m.H * n, n)
        before = m.K.copy(), m.V.copy(), None if m.bias is None else m.bias.copy()
        # (a request whose indices pass the ones given is refused: it asks for more cells than there are)
        ask = [int(s) if cu[i + 1] <= total else -1 for i, s in enumerate(seqs)]
        want = m.compact(ask, start, cu, good, v, beta)
        for l, k in bad:
            i = int(np.searchsorted(cu[1:], k, side="right"))
            p, x = m.spots(m.table[seqs[i]], [start[i] + k - cu[i]])
            m.K[l, p, x], m.V[l, p, x] = before[0][l, p, x], before[1][l, p, x]
            if m.bias is not None:
                m.bias[l, p, :, x] = before[2][l, p, :, x]
        rc = self.dll.kvc_cache_compact(self.c, len(seqs), bufs[0].value, bufs[1].value, bufs[2].value, total,
                                        bufs[3].value, n, ctypes.byref(pv) if pv else None,
                                        ctypes.byref(pb) if pb else None, bufs[4].value, *self.ws(len(seqs)), None)
        self._status(rc, want, bufs[4], what)


@pytest.mark.parametrize("values", [False, True])
@pytest.mark.parametrize("betas", [False, True])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("kt", [F16, Q8_0])
def test_indices_that_do_not_fit(dll, kt, shared, betas, values):   # noqa: F811
    # negative, past the end, below their place: the cell is left as it was, in place and on a fresh page
    c = BadIndices(dll, seed=3, pages=24, page=16, max_pages=10, L=2, k_type=kt, v_type=kt)
    c.extend([0], [100])
    c.write([0], [100])
    if shared:
        c.fork([0], [1])
    start = 5
    idx = np.stack([np.sort(c.rng.choice(np.arange(1, 95), 40, replace=False)) for _ in range(2)])
    bad = [(0, 3), (0, 39), (1, 0), (1, 17), (1, 38)]
    for (l, k), x in zip(bad, (-1, 95, -(1 << 31), 16, (1 << 31) - 1)):
        idx[l, k] = x
    c.run([0], [start], [0, 40], idx, 40, values, betas, bad, f"shared={shared}")


def test_fewer_indices_than_asked_for(dll):   # noqa: F811
    # a request whose last index is past n_idx is refused; the ones before it are done
    c = BadIndices(dll, seed=4, pages=24, page=16, max_pages=10, L=2)
    c.extend([0, 1, 2], [60, 50, 40])
    c.write([0, 1, 2], [60, 50, 40])
    cu = [0, 20, 35, 45]
    idx = np.concatenate([np.stack([c.some(n, k) for _ in range(2)]) for n, k in ((60, 20), (50, 15), (40, 10))], 1)
    c.run([0, 1, 2], [0, 0, 0], cu, idx, 34, what="34 of 45")
    assert c.m.len.tolist()[:3] == [20, 50, 40]
    c.run([1, 2], [0, 0], [0, 15, 25], idx[:, 20:], 25, True, True, what="all of them")


@pytest.mark.parametrize("kt,H,dk,dv", [(F16, 1, 33, 5), (BF16, 3, 7, 9), (F16, 2, 32, 64), (Q8_0, 1, 32, 5), (Q8_0, 3, 96, 8)])
def test_keys_and_values_of_different_types(dll, kt, H, dk, dv):   # noqa: F811
    # rows of K whose bytes are no multiple of 4 beside F32 values
    c = Cache(dll, seed=6, pages=40, page=16, max_pages=16, L=2, H=H, dk=dk, dv=dv, k_type=kt, v_type=F32)
    c.extend([0, 1], [70, 90])
    c.fork([1], [2])
    kept = [c.some(70, 30) for _ in range(2)], [c.some(80, 31) for _ in range(2)]
    c.compact([0, 2], [0, 10], kept, values=True, betas=True)
    c.compact([1], [3], [[c.some(87, 40) for _ in range(2)]], values=True, heads_apart=True)


def test_rows_before_the_first_sequence(dll):   # noqa: F811
    # cu need not begin at 0: rows and indices before it belong to no request
    c = BadIndices(dll, seed=9, pages=24, page=16, max_pages=10, L=2)
    c.extend([0, 1], [60, 50])
    c.write([0, 1], [60, 50])
    rows = [c.rng.integers(0, 256, (2, 12, 128), np.uint8) for _ in range(2)]
    bufs = [dev(x) for x in rows]
    a, cu = dev(np.int32([1, 0])), np.int32([4, 7, 10])
    r, dcu = [kc.Rows(b.value, 12 * 128, 128) for b in bufs], dev(cu)
    assert dll.kvc_cache_write(c.c, 0, 2, 2, a.value, dcu.value, 10, F16, *r, None) == 0
    c.m.write(0, 2, [1, 0], cu, *rows)
    c.check("write from row 4 on")
    idx = np.concatenate([np.full((2, 5), -7), np.stack([c.some(60, 20) for _ in range(2)]), np.stack([c.some(50, 9) for _ in range(2)])], 1)
    c.run([0, 1], [0, 0], [5, 25, 34], idx, 34, True, True, what="indices from the sixth on")
