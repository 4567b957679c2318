"""A cache kept to a budget as a server does it (include/kvc-cache.h): prompts and tokens under a window, the weights
they give gathered, cells picked by them, the cache compacted and the weights moved along; captured into a graph, on
streams side by side, refused in part, and past 4 GiB."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from budget_model import window_seen
from cache_model import BF16, F16, F32, Q8_0, attend, bf16, decode, encode
from kvc_harness import kc
from test_gpu_cache_attn import Strided, compare, wide
from test_gpu_cache_run import Server, _graph_api, dev, lib   # noqa: F401 (the fixture)
from test_gpu_evict import picked, scores
from test_gpu_weigh import weights_of

pytestmark = pytest.mark.gpu


class Budget(Server):
    """A server's cache with the weights its cells gather."""

    def __init__(self, dll, L, pages, page, seqs, max_pages, H, d, typ, qt, first, last):
        super().__init__(dll, L, pages, page, seqs, max_pages, H, d, typ, bias=False)
        self.qt, self.first, self.last, self.seqs, self.room = qt, first, last, seqs, max_pages * page
        self.w = dev(np.full((L, seqs, H, self.room), np.nan, np.float32))   # (every cell begins with its own token)
        self.granted, self.cu = dev(np.zeros(16, np.int32)), dev(np.zeros(17, np.int32))
        self.window = kc.Window(first, last)

    def weights(self):
        return self.w.download(np.float32, self.L * self.seqs * self.H * self.room).reshape(self.L, self.seqs, self.H, self.room)

    def rows(self, layer, seq, n):
        _, _, k, v, _ = self.read(seq, n)
        return k[layer], v[layer]

    def step(self, layer, q, seqs, news, decay, tail=0, mask=None):
        """Attention under the window and the weights it gives, of tokens whose cells are the last ones."""
        cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        n, Hq, d = q.shape
        sq, so = Strided(q, self.qt), Strided(np.zeros((n, Hq, d)), self.qt)
        lse = dev(np.zeros((n, Hq), np.float32))
        a = kc.CacheAttnArgs(q=sq.heads(), o=so.heads(), lse=lse.value, seqs=self.arr(np.int32(seqs)), cu=self.arr(cu),
                             mask=self.arr(mask) if mask is not None else None, mask_words=1, layer=layer, type=self.qt,
                             n_seq=len(seqs), n_tok=n, n_head=Hq, max_new=max(news), max_len=self.room)
        size = self.dll.kvc_attn_cache_window_workspace(self.c, a, self.window)
        ws = dev(np.zeros(max(size, 16), np.uint8))
        self.ok(self.dll.kvc_attn_cache_window(self.c, a, self.window, ws.value, size, None))
        self.ok(self.dll.kvc_cache_weigh(self.c, a, self.window, kc.WeighArgs(self.w.value, decay, tail, 0), None))
        return so.read()[0], lse.download(np.float32, n * Hq).reshape(n, Hq), wide(sq._view(sq.host), self.qt)

    def evict(self, seqs, start, keep, recent, max_len=None, shared=False):
        """pick, compact, move the weights: returns granted, cu and the indices [layers][..]"""
        n = len(seqs)
        n_idx = sum(keep)
        idx = dev(np.full(self.L * n_idx, -1, np.int32))
        s, st, kp = (self.arr(np.int32(x)) for x in (seqs, start, keep))
        ld = 0 if shared else n_idx
        a = kc.PickArgs(seqs=s, start=st, keep=kp, weight=self.w.value, idx=idx.value, ld_idx=ld, cu=self.cu.value,
                        granted=self.granted.value, status=self.status.value, n_idx=n_idx, recent=recent,
                        heads=kc.HEADS_SUM, max_len=self.room if max_len is None else max_len)
        size = self.dll.kvc_cache_pick_workspace(self.c, n, a)
        ws = dev(np.zeros(size + 16, np.uint8))
        self.ok(self.dll.kvc_cache_pick(self.c, n, a, ws.value, size, None))
        self.ok(self.dll.kvc_cache_compact(self.c, n, self.granted.value, st, self.cu.value, n_idx, idx.value, ld, None, None,
                                           self.status.value, self.ws.value, self.size, None))
        self.ok(self.dll.kvc_cache_take_weights(self.c, n, self.granted.value, self.granted.value, st, self.cu.value, n_idx,
                                                idx.value, ld, self.status.value, self.w.value, None))
        self.keep += [idx, ws]
        return (self.granted.download(np.int32, n).tolist(), self.cu.download(np.int32, n + 1).tolist(),
                idx.download(np.int32, self.L * n_idx).reshape(self.L, n_idx))


@pytest.mark.parametrize("typ,qt", [(F32, F32), (F16, F16), (BF16, BF16), (Q8_0, BF16)])
def test_a_chat_under_a_budget(lib, typ, qt):   # noqa: F811
    """Two prompts, tokens until a budget is passed, eviction, more tokens, a sample of one of them that drafts a tree and
    is evicted for itself: every result is that of what the cache then holds."""
    dll = lib.dll
    L, H, G, d, page, first, last, budget = 2, 2, 2, 64, 16, 4, 48, 64
    rng = np.random.default_rng(11)
    s = Budget(dll, L, 90, page, 4, 20, H, d, typ, qt, first, last)
    held, lens = {}, [150, 37]
    weight = {}                                             # seq -> [L][H][cells], and how far each may be off
    tol = {}

    def new_rows(n):
        return [decode(encode(rng.standard_normal((L, n, H * d)).astype(np.float32), typ), typ).reshape(L, n, H, d) for _ in range(2)]

    def attended(seqs, news, decay, tail=0, mask=None, see=None):
        for l in range(L):
            q = rng.standard_normal((sum(news), H * G, d))
            o, lse, qd = s.step(l, q, seqs, news, decay, tail, mask)
            at = 0
            for b, n in zip(seqs, news):
                k, v = held[b][0][l], held[b][1][l]
                seen = window_seen(len(k), n, first, last, see)
                want = attend(qd[at:at + n], k, v, seen, None, d ** -0.5, qt)
                compare(o[at:at + n], lse[at:at + n].astype(float), want, qt, f"layer {l}, sequence {b}")
                w, t = weights_of(qd[at:at + n], k, None, seen, d ** -0.5, lse[at:at + n].astype(float), tail)
                old = np.zeros((H, len(k)))
                m = len(k) - n
                if decay:
                    old[:, :m] = decay * weight[b][l][:, :m]
                    t[:, :m] += decay * tol[b][l][:, :m]
                weight[b][l], tol[b][l] = old + w, t + 2.0 ** -22 * old
                at += n
        got = s.weights()
        for b in seqs:
            for l in range(L):
                off = np.abs(got[l, b, :, :weight[b][l].shape[1]] - weight[b][l])
                assert (off <= tol[b][l]).all(), f"weights of layer {l}, sequence {b}"

    def grow(seqs, news):
        k, v = new_rows(sum(news))
        s.extend(seqs, news)
        for l in range(L):
            s.write(l, seqs, news, k[l], v[l])
        at = 0
        for b, n in zip(seqs, news):
            old = held.get(b, (k[:, :0], v[:, :0]))
            held[b] = [np.concatenate([x, y[:, at:at + n]], 1) for x, y in zip(old, (k, v))]
            at += n

    def evicted(seqs, start, keep, recent, shared=False):
        w = s.weights()
        granted, cu, idx = s.evict(seqs, start, keep, recent, shared=shared)
        assert granted == list(seqs)
        for i, b in enumerate(seqs):
            n = held[b][0].shape[1]
            for l in range(L):
                rows = w[:, b].reshape(-1, s.room) if shared else w[l, b]
                want = picked(scores(rows, False), start[i], n, keep[i], recent)
                pick = idx.reshape(-1)[:sum(keep)][None] if shared else idx
                assert pick[0 if shared else l, cu[i]:cu[i + 1]].tolist() == want.tolist(), f"cells of layer {l}, sequence {b}"
                cells = np.r_[0:start[i], start[i] + want]
                weight[b][l], tol[b][l] = weight[b][l][:, cells], tol[b][l][:, cells]
                new = [x[l][cells] for x in held[b]]
                held.setdefault(("new", b), []).append(new)
            held[b] = [np.stack([x[j] for x in held[("new", b)]]) for j in range(2)]
            del held[("new", b)]
            kd, vd = s.read(b, held[b][0].shape[1])[2:4]
            assert np.array_equal(kd, held[b][0]) and np.array_equal(vd, held[b][1]), f"rows of sequence {b}"
            got = s.weights()
            for l in range(L):
                assert np.array_equal(got[l, b, :, :len(kd[l])], w[l, b][:, np.r_[0:start[i], start[i] + idx.reshape(-1)[:sum(keep)][cu[i]:cu[i + 1]]]]
                                      if shared else w[l, b][:, np.r_[0:start[i], start[i] + idx[l, cu[i]:cu[i + 1]]]]), "weights moved"

    # prompts: the same rows by the packed form and through the cache
    grow([0, 2], lens)
    for b in (0, 2):
        weight[b], tol[b] = [None] * L, [None] * L
    attended([0, 2], lens, 0.0, tail=16)
    if typ == qt:
        for b, n in ((0, lens[0]), (2, lens[1])):
            q = rng.standard_normal((n, H * G, d))
            sq, sk, sv, so = (Strided(x, qt) for x in (q, held[b][0][0], held[b][1][0], np.zeros((n, H * G, d))))
            lse = dev(np.zeros((n, H * G), np.float32))
            s.ok(dll.kvc_attn_prompt_window(kc.PromptArgs(q=sq.heads(), k=sk.heads(), v=sv.heads(), o=so.heads(), lse=lse.value,
                                                          cu=s.arr(np.int32([0, n])), type=qt, n_seq=1, n_tok=n, n_head=H * G,
                                                          n_head_kv=H, d_k=d, d_v=d), s.window, None))
            want = attend(wide(sq._view(sq.host), qt), held[b][0][0], held[b][1][0], window_seen(n, n, first, last), None, d ** -0.5, qt)
            compare(so.read()[0], lse.download(np.float32, n * H * G).reshape(n, -1).astype(float), want, qt, "packed prompt")
    evicted([0, 2], [first, first], [budget - first, budget - first], 16)
    assert s.len.download(np.int32, 4).tolist() == [64, 0, 37, 0]
    for _ in range(3):
        grow([0, 2], [1, 1])
        attended([0, 2], [1, 1], 1.0)
    evicted([0], [first], [budget - first], 16, shared=True)
    # a sample of sequence 0 goes its own way: a tree of drafts, some accepted, evicted again; 0 stays as it is
    s.ok(dll.kvc_cache_fork(s.c, 1, s.arr(np.int32([0])), s.arr(np.int32([3])), s.status.value, None))
    s.ok(dll.kvc_cache_take_weights(s.c, 1, s.arr(np.int32([0])), s.arr(np.int32([3])), None, None, 0, None, 0, s.status.value,
                                    s.w.value, None))
    held[3], weight[3], tol[3] = [x.copy() for x in held[0]], [x.copy() for x in weight[0]], [x.copy() for x in tol[0]]
    before = s.weights()[:, 0, :, :64].copy()
    grow([3], [5])
    see = np.array([[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 0, 1, 0, 0], [1, 1, 0, 1, 0], [1, 0, 0, 0, 1]], bool)
    attended([3], [5], 0.9375, mask=np.uint64([1, 3, 5, 11, 17]), see=see)
    evicted([3], [first], [40], 8)
    kd, vd = s.read(0, 64)[2:4]
    assert np.array_equal(kd, held[0][0]) and np.array_equal(vd, held[0][1])
    assert np.array_equal(s.weights()[:, 0, :, :64], before)
    grow([0, 3], [2, 1])
    attended([0, 3], [2, 1], 1.0)


def test_captured_steps(lib):   # noqa: F811
    """Reserve, write, attend under a window, weigh, pick, compact and move the weights in a graph, replayed with other rows
    and queries between eager calls: every replay is the eager result."""
    import hiprt
    dll, h = lib.dll, _graph_api()
    H, G, d, page, first, last = 2, 2, 64, 16, 2, 700
    rng = np.random.default_rng(3)
    s = Budget(dll, 1, 160, page, 2, 70, H, d, F16, F16, first, last)
    lens, news, n = [1000, 337], [3, 2], 5
    s.extend([0, 1], lens)
    s.write(0, [0, 1], lens, *(rng.standard_normal((sum(lens), H, d)) for _ in range(2)))
    rows = [dev(np.zeros(n * s.rb, np.uint8)) for _ in range(2)]
    q, o = (dev(np.zeros((n, H * G, d), np.float16)) for _ in range(2))
    lse = dev(np.zeros((n, H * G), np.float32))
    seqs, cu, count, start, keep = (s.arr(np.int32(x)) for x in ([0, 1], [0, 3, 5], news, [2, 2], [990, 300]))
    n_idx = 1290
    idx = dev(np.zeros(n_idx, np.int32))
    granted = dev(np.zeros(2, np.int32))
    a = kc.CacheAttnArgs(q=kc.Heads(q.value, H * G * d, d), o=kc.Heads(o.value, H * G * d, d), lse=lse.value,
                         seqs=granted.value, cu=cu, n_seq=2, n_tok=n, n_head=H * G, max_new=3, max_len=1020, type=F16)
    size = dll.kvc_attn_cache_window_workspace(s.c, a, s.window)
    assert size > 0     # (a call of two kernels)
    ws = dev(np.zeros(size, np.uint8))
    pa = kc.PickArgs(seqs=seqs, start=start, keep=keep, weight=s.w.value, idx=idx.value, ld_idx=n_idx, cu=s.cu.value,
                     granted=s.granted.value, status=s.status.value, n_idx=n_idx, recent=9, heads=kc.HEADS_SUM, max_len=1020)
    psize = dll.kvc_cache_pick_workspace(s.c, 2, pa)
    pws = dev(np.zeros(psize, np.uint8))
    w0 = np.exp(rng.standard_normal((1, 2, H, s.room))).astype(np.float32)
    state = [(s.K, s.K.download(np.uint8, s.K.nbytes)), (s.V, s.V.download(np.uint8, s.V.nbytes)),
             (s.table, s.table.download(np.int32, 140)), (s.len, s.len.download(np.int32, 2)), (s.refs, s.refs.download(np.int32, 160)), (s.w, w0)]

    def step(st):
        s.ok(dll.kvc_cache_extend_granted(s.c, 2, seqs, count, s.status.value, granted.value, s.ws.value, s.size, st))
        r = [kc.Rows(x.value, 0, s.rb) for x in rows]
        s.ok(dll.kvc_cache_write(s.c, 0, 1, 2, granted.value, cu, n, F16, r[0], r[1], st))
        s.ok(dll.kvc_attn_cache_window(s.c, a, s.window, ws.value, size, st))
        s.ok(dll.kvc_cache_weigh(s.c, a, s.window, kc.WeighArgs(s.w.value, 0.9375, 0, 0), st))
        s.ok(dll.kvc_cache_pick(s.c, 2, pa, pws.value, psize, st))
        s.ok(dll.kvc_cache_compact(s.c, 2, s.granted.value, start, s.cu.value, n_idx, idx.value, n_idx, None, None, s.status.value,
                                   s.ws.value, s.size, st))
        s.ok(dll.kvc_cache_take_weights(s.c, 2, s.granted.value, s.granted.value, start, s.cu.value, n_idx, idx.value, n_idx,
                                        s.status.value, s.w.value, st))

    def result(i, run):
        r = np.random.default_rng(100 + i)
        for buf, x in state:
            buf.upload(x)
        for x in rows:
            x.upload(encode(r.standard_normal((n, H * d)), F16))
        q.upload(r.standard_normal((n, H * G, d)).astype(np.float16))
        run()
        hiprt.synchronize()
        return [o.download(np.uint16, n * H * G * d), lse.download(np.uint32, n * H * G), s.len.download(np.int32, 2),
                idx.download(np.int32, n_idx), s.weights().view(np.uint32), s.K.download(np.uint8, s.K.nbytes)]

    stream = ctypes.c_void_p()
    hiprt.check(h.hipStreamCreate(ctypes.byref(stream)))
    graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
    hiprt.check(h.hipStreamBeginCapture(stream, 2))
    step(stream)
    hiprt.check(h.hipStreamEndCapture(stream, ctypes.byref(graph)))
    hiprt.check(h.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0))
    for i in range(4):
        want = result(i, lambda: step(None))
        got = result(i, lambda: hiprt.check(h.hipGraphLaunch(exe, stream)))
        for x, y in zip(want, got):
            assert np.array_equal(x, y), f"replay {i}"
        assert want[2].tolist() == [992, 302]
    hiprt.check(h.hipGraphExecDestroy(exe))
    hiprt.check(h.hipGraphDestroy(graph))
    hiprt.check(h.hipStreamDestroy(stream))


def test_calls_at_once(lib):   # noqa: F811
    """Windows, weights and picks of two layers on two streams, each with arrays and a workspace of its own."""
    import hiprt
    dll, h = lib.dll, _graph_api()
    H, G, d, page, n_seq = 4, 2, 128, 32, 4
    rng = np.random.default_rng(9)
    s = Server(dll, 2, 300, page, n_seq, 70, H, d, BF16, bias=False)
    lens = [2000, 1500, 900, 64]
    s.extend(range(n_seq), lens)
    for l in range(2):
        s.write(l, range(n_seq), lens, *(rng.standard_normal((sum(lens), H, d)) for _ in range(2)))
    hiprt.synchronize()
    cu, room = s.arr(np.int32([0, 1, 2, 3, 4])), 70 * page
    start, keep, seqs = (s.arr(np.int32(x)) for x in ([4] * 4, [700, 500, 300, 60], [0, 1, 2, 3]))
    calls, streams = [], []
    for l in range(2):
        q, o = dev(bf16(rng.standard_normal((4, H * G, d)))), dev(np.zeros((4, H * G, d), np.uint16))
        lse, w = dev(np.zeros((4, H * G), np.float32)), dev(np.zeros((2, n_seq, H, room), np.float32))
        a = kc.CacheAttnArgs(q=kc.Heads(q.value, H * G * d, d), o=kc.Heads(o.value, H * G * d, d), lse=lse.value, cu=cu, layer=l,
                             type=BF16, n_seq=4, n_tok=4, n_head=H * G, max_new=1, max_len=2000)
        out = [dev(np.zeros(k, np.int32)) for k in (2 * 1560, 5, 4, 4)]
        p = kc.PickArgs(seqs=seqs, start=start, keep=keep, weight=w.value, idx=out[0].value, ld_idx=1560, cu=out[1].value,
                        granted=out[2].value, status=out[3].value, n_idx=1560, recent=5, heads=kc.HEADS_SUM, max_len=2000)
        win = kc.Window(4, 1500)
        sizes = dll.kvc_attn_cache_window_workspace(s.c, a, win), dll.kvc_cache_pick_workspace(s.c, 4, p)
        ws = [dev(np.zeros(max(k, 16), np.uint8)) for k in sizes]
        st = ctypes.c_void_p()
        hiprt.check(h.hipStreamCreate(ctypes.byref(st)))
        calls.append((a, p, win, q, o, lse, w, out, ws, sizes))
        streams.append(st)

    def one(i, st):
        a, p, win, _, _, _, w, _, ws, sizes = calls[i]
        s.ok(dll.kvc_attn_cache_window(s.c, a, win, ws[0].value, sizes[0], st))
        s.ok(dll.kvc_cache_weigh(s.c, a, win, kc.WeighArgs(w.value, 0.0, 0, 0), st))
        s.ok(dll.kvc_cache_pick(s.c, 4, p, ws[1].value, sizes[1], st))

    def got(i):
        a, p, win, _, o, _, w, out, _, _ = calls[i]
        return o.download(np.uint16, 4 * H * G * d).tobytes(), out[0].download(np.int32, 2 * 1560).tobytes(), w.download(np.uint8, w.nbytes).tobytes()
    alone = []
    for i in range(2):
        one(i, None)
        hiprt.synchronize()
        alone.append(got(i))
        calls[i][4].zero()
        calls[i][7][0].zero()
    hiprt.synchronize()
    for _ in range(20):
        for i in range(2):
            one(i, streams[i])
    hiprt.synchronize()
    for i in range(2):
        assert alone[i] == got(i)
        hiprt.check(h.hipStreamDestroy(streams[i]))
    assert alone[0] != alone[1]


def test_refused_in_part(lib):   # noqa: F811
    """Of three requests one names no sequence and one a sequence longer than the call was told of: those keep all their
    cells and weights, the third is evicted."""
    dll = lib.dll
    H, d, page = 2, 64, 16
    rng = np.random.default_rng(5)
    s = Budget(dll, 1, 60, page, 3, 20, H, d, F32, F32, 0, 10)
    s.extend([0, 1, 2], [300, 100, 50])
    s.write(0, [0, 1, 2], [300, 100, 50], *(rng.standard_normal((450, H, d)) for _ in range(2)))
    w = rng.random((1, 3, H, s.room)).astype(np.float32)
    s.w.upload(w)
    k0 = [s.read(b, n)[2] for b, n in ((0, 300), (1, 100), (2, 50))]
    granted, cu, idx = s.evict([0, 7, 1], [0, 0, 3], [20, 20, 20], 4, max_len=128)
    assert granted == [-1, -1, 1] and cu == [0, 0, 0, 20]
    assert s.status.download(np.int32, 3).tolist() == [kc.REQ_BAD, kc.REQ_BAD, 0]
    assert s.len.download(np.int32, 3).tolist() == [300, 23, 50]
    cells = np.r_[0:3, 3 + idx[0, :20]]
    assert np.array_equal(s.read(0, 300)[2], k0[0]) and np.array_equal(s.read(2, 50)[2], k0[2])
    assert np.array_equal(s.read(1, 23)[2], k0[1][:, cells])
    got = s.weights()
    assert np.array_equal(got[:, [0, 2]], w[:, [0, 2]]) and np.array_equal(got[0, 1, :, :23], w[0, 1][:, cells])


@pytest.mark.parametrize("new", [1, 12, 40])
def test_offsets_past_32_bits(lib, new):   # noqa: F811
    """The last layer of a cache of more than 4 GiB, its last pages, and weights whose rows stand past 4 GiB."""
    import hiprt
    dll = lib.dll
    H, G, d, page, pages, max_pages = 8, 4, 128, 1024, 1100, 1 << 16
    if hiprt.mem_free() < 24 << 30:
        pytest.skip("not enough device memory")
    L, rb, room = 2, 2 * H * d, (1 << 16) * 1024
    K = hiprt.DevBuf(L * pages * page * rb)
    W = hiprt.DevBuf(4 * L * 2 * H * room)       # 8 GiB
    assert K.nbytes > 1 << 32 and W.nbytes > 1 << 32
    K.zero()
    last, n = [pages - 1, pages - 2], 2 * page
    rng = np.random.default_rng(new)
    k, v = (bf16(rng.standard_normal((n, H, d))) for _ in range(2))
    V = hiprt.DevBuf(L * pages * page * rb)
    V.zero()
    for i, p in enumerate(last):
        at = ((L - 1) * pages + p) * page * rb
        K.upload(k[i * page:(i + 1) * page], at)
        V.upload(v[i * page:(i + 1) * page], at)
    table = np.full((2, max_pages), -1, np.int32)
    table[1, :2] = last
    bufs = [dev(x) for x in (table, np.int32([0, n]), np.int32([0] * (pages - 2) + [1, 1]))]
    c = kc.KvCache(n_layers=L, n_pages=pages, page_size=page, max_seqs=2, max_pages=max_pages, n_head_kv=H, d_k=d, d_v=d, k_type=BF16,
                   v_type=BF16, K=K.value, V=V.value, table=bufs[0].value, len=bufs[1].value, refs=bufs[2].value)
    q, o = Strided(rng.standard_normal((new, H * G, d)), BF16), Strided(np.zeros((new, H * G, d)), BF16)
    lse, cu, seqs = dev(np.zeros((new, H * G), np.float32)), dev(np.int32([0, new])), dev(np.int32([1]))
    a = kc.CacheAttnArgs(q=q.heads(), o=o.heads(), lse=lse.value, seqs=seqs.value, cu=cu.value, layer=L - 1, type=BF16, n_seq=1,
                         n_tok=new, n_head=H * G, max_new=new, max_len=n)
    win = kc.Window(100, 600)
    size = dll.kvc_attn_cache_window_workspace(c, a, win)
    ws = dev(np.zeros(max(size, 16), np.uint8))
    assert dll.kvc_attn_cache_window(c, a, win, ws.value, size, None) == 0
    f = lambda x: decode(x.view(np.uint8).reshape(n, -1), BF16).reshape(n, H, d)  # noqa: E731
    seen, qd = window_seen(n, new, 100, 600), wide(q._view(q.host), BF16)
    want = attend(qd, f(k), f(v), seen, None, d ** -0.5, BF16)
    l = lse.download(np.float32, new * H * G).reshape(new, -1)
    compare(o.read()[0], l.astype(float), want, BF16, f"{new} new")
    assert dll.kvc_cache_weigh(c, a, win, kc.WeighArgs(W.value, 0.0, 0, 0), None) == 0
    row = lambda layer, h: W.download(np.float32, n, 4 * (((layer * 2 + 1) * H + h) * room))  # noqa: E731
    w, tol = weights_of(qd, f(k), None, seen, d ** -0.5, l.astype(float), 0)
    got = np.stack([row(L - 1, h) for h in range(H)])
    assert (np.abs(got - w) <= tol).all()
    # layer 0's rows, then the pick and the move over both
    for h in range(H):
        W.upload(np.arange(n, dtype=np.float32)[::-1], 4 * ((0 * 2 + 1) * H + h) * room)
    start, keep, idx, out = dev(np.int32([5])), dev(np.int32([50])), dev(np.zeros((2, 50), np.int32)), [dev(np.zeros(2, np.int32)) for _ in range(3)]
    p = kc.PickArgs(seqs=seqs.value, start=start.value, keep=keep.value, weight=W.value, idx=idx.value, ld_idx=50, cu=out[0].value,
                    granted=out[1].value, status=out[2].value, n_idx=50, recent=10, heads=kc.HEADS_SUM, max_len=n)
    psize = dll.kvc_cache_pick_workspace(c, 1, p)
    pws = dev(np.zeros(psize, np.uint8))
    assert dll.kvc_cache_pick(c, 1, p, pws.value, psize, None) == 0
    ii = idx.download(np.int32, 100).reshape(2, 50)
    assert ii[0].tolist() == list(range(40)) + list(range(n - 15, n - 5))
    assert ii[1].tolist() == picked(scores(got, False), 5, n, 50, 10).tolist()
    assert dll.kvc_cache_take_weights(c, 1, seqs.value, seqs.value, start.value, out[0].value, 50, idx.value, 50, out[2].value, W.value, None) == 0
    for h in range(H):
        assert np.array_equal(row(L - 1, h)[:55], got[h][np.r_[0:5, 5 + ii[1]]])
