"""The paged cache as a server uses it (include/kvc-cache.h): prompts, pages,
compaction and drafts one after another, two calls at once, and captured into
HIP graphs that are replayed with other data."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from cache_model import BF16, F16, F32, Q8_0, attend, bf16, decode, encode, row_bytes
from kvc_harness import kc
from test_gpu_cache_attn import Strided, compare, typed, wide

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    lib = kc.load_product()
    if not lib.dll.kv_compact_hip_available():
        pytest.fail("no usable GPU for the GPU test tier")
    kc.bind_device_api(lib.dll)
    kc.bind_cache(lib.dll)
    return lib


def dev(x):
    import hiprt
    x = np.ascontiguousarray(x)
    b = hiprt.DevBuf(max(x.nbytes, 16))
    if x.nbytes:
        b.upload(x)
    return b


class Server:
    """A cache of L layers on the device, filled with what no one may read."""

    def __init__(self, dll, L, pages, page, seqs, max_pages, H, d, typ, bias=True):
        self.dll, self.L, self.page, self.H, self.d, self.typ = dll, L, page, H, d, typ
        rb = row_bytes(typ, H * d)
        self.rb, self.pages, self.max_pages = rb, pages, max_pages
        junk = np.full(L * pages * page * rb, 0xFF, np.uint8)
        self.K, self.V = dev(junk), dev(junk)
        self.bias = dev(np.full(L * pages * H * page, np.nan, np.float32)) if bias else None
        self.table, self.len, self.refs = (dev(np.full(n, 7, np.int32)) for n in (seqs * max_pages, seqs, pages))
        self.c = kc.KvCache(n_layers=L, n_pages=pages, page_size=page, max_seqs=seqs, max_pages=max_pages, n_head_kv=H,
                            d_k=d, d_v=d, k_type=typ, v_type=typ, K=self.K.value, V=self.V.value,
                            bias=self.bias.value if bias else None, table=self.table.value, len=self.len.value,
                            refs=self.refs.value)
        self.size = dll.kvc_cache_workspace(self.c, 16)
        self.ws = dev(np.zeros(self.size, np.uint8))
        self.status = dev(np.zeros(16, np.int32))
        self.keep = []
        self.ok(dll.kvc_cache_reset(self.c, None))

    def ok(self, rc):
        assert rc == 0, rc

    def arr(self, x):
        self.keep.append(dev(x))
        return self.keep[-1].value

    def done(self, n):
        assert self.status.download(np.int32, n).tolist() == [0] * n

    def extend(self, seqs, counts):
        self.ok(self.dll.kvc_cache_extend(self.c, len(seqs), self.arr(np.int32(seqs)), self.arr(np.int32(counts)),
                                          self.status.value, self.ws.value, self.size, None))
        self.done(len(seqs))

    def write(self, layer, seqs, counts, k, v):
        """k, v fp32 values of the cache's type [rows][H][d]"""
        cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        rows = [encode(x.reshape(len(x), -1), self.typ) for x in (k, v)]
        r = [kc.Rows(self.arr(x), 0, self.rb) for x in rows]
        self.ok(self.dll.kvc_cache_write(self.c, layer, 1, len(seqs), self.arr(np.int32(seqs)), self.arr(cu), int(cu[-1]),
                                         self.typ, r[0], r[1], None))

    def read(self, seq, n):
        k, v = (dev(np.zeros(self.L * n * self.rb, np.uint8)) for _ in range(2))
        b = dev(np.zeros(self.L * self.H * n, np.float32))
        self.ok(self.dll.kvc_cache_read(self.c, seq, 0, n, k.value, v.value, b.value if self.bias else None, None))
        out = [decode(x.download(np.uint8, self.L * n * self.rb).reshape(self.L, n, -1), self.typ).reshape(
            self.L, n, self.H, self.d) for x in (k, v)]
        return k, v, out[0], out[1], b.download(np.float32, self.L * self.H * n).reshape(self.L, self.H, n)

    def attend(self, layer, q, typ, seqs, news, mask=None, words=1, max_len=4096):
        cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        n, Hq, d = q.shape
        sq, so = Strided(q, typ), Strided(np.zeros((n, Hq, d)), typ)
        lse = dev(np.zeros((n, Hq), np.float32))
        a = kc.CacheAttnArgs(q=sq.heads(), o=so.heads(), lse=lse.value, seqs=self.arr(np.int32(seqs)), cu=self.arr(cu),
                             mask=self.arr(mask) if mask is not None else None, mask_words=words, layer=layer, type=typ,
                             n_seq=len(seqs), n_tok=n, n_head=Hq, max_new=max(news), max_len=max_len)
        size = self.dll.kvc_attn_cache_workspace(self.c, a)
        ws = dev(np.zeros(max(size, 16), np.uint8))
        self.ok(self.dll.kvc_attn_cache(self.c, a, ws.value, size, None))
        return so.read()[0], lse.download(np.float32, n * Hq).reshape(n, Hq), wide(sq._view(sq.host), typ)


@pytest.mark.parametrize("typ", [F32, F16, BF16])
def test_prompt_compaction_and_drafts(lib, typ):
    """A prompt is computed and stored, its cache compacted with the library's own compaction, shared, drafted on, and
    the accepted drafts kept: each attention is the one of what the cache then holds."""
    dll = lib.dll
    L, H, G, d, page, T = 2, 2, 2, 64, 32, 700
    rng = np.random.default_rng(5)
    s = Server(dll, L, 80, page, 4, 40, H, d, typ)
    k, v = (rng.standard_normal((L, T, H, d)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((L, T, H * G, d)).astype(np.float32)
    k, v = (decode(encode(x.reshape(L, T, -1), typ), typ).astype(np.float32).reshape(L, T, H, d) for x in (k, v))
    s.extend([1], [T])
    for l in range(L):
        sq, sk, sv, so = (Strided(x, typ) for x in (q[l], k[l], v[l], np.zeros((T, H * G, d))))
        lse = dev(np.zeros((T, H * G), np.float32))
        s.ok(dll.kvc_attn_prompt(kc.PromptArgs(q=sq.heads(), k=sk.heads(), v=sv.heads(), o=so.heads(), lse=lse.value,
                                               cu=s.arr(np.int32([0, T])), type=typ, n_seq=1, n_tok=T, n_head=H * G,
                                               n_head_kv=H, d_k=d, d_v=d), None))
        s.write(l, [1], [T], k[l], v[l])
        if l == 0:
            want = attend(wide(sq._view(sq.host), typ)[-40:], k[0].astype(float), v[0].astype(float),
                          np.tril(np.ones((T, T), bool))[-40:], None, d ** -0.5, typ)
            compare(so.read()[0][-40:], lse.download(np.float32, T * H * G).reshape(T, -1)[-40:].astype(float), want, typ,
                    "prompt")
    # compaction: rows as the cache holds them, beta fitted
    kb, vb, kd, vd, b = s.read(1, T)
    assert np.array_equal(kd, k) and np.array_equal(vd, v) and not b.any()
    p = lib.params(target_ratio=0.2, skip_beta=0, use_cheap_qref=1)
    t, _ = kc.plan(dll, T, 0, False, p)
    idx, beta, cv, st = (dev(np.zeros(n, np.float32)) for n in (L * t, L * H * t, L * H * t * d, L * 3))
    out = kc.DeviceOut(idx.value, beta.value, cv.value, st.value)
    if typ == F32:
        s.ok(dll.kvc_compact_layers_device(kb.value, vb.value, None, L, T, 0, H, d, d, T * H * d, T * H * d, 0, p, None, out, None))
        vals = kc.Values(cv.value, 4 * H * t * d, 4 * d, 4 * t * d)
    else:
        ko, vo = (dev(np.zeros(L * t * s.rb, np.uint8)) for _ in range(2))
        s.ok(dll.kvc_compact_quantized_layers_device(kb.value, vb.value, None, L, typ, typ, s.rb, s.rb, T, 0, H, d, d,
                                                     T * s.rb, T * s.rb, 0, p, out, ko.value, vo.value, None))
        vals = kc.Values(vo.value, t * s.rb, s.rb, s.rb // H)
    s.ok(dll.kvc_cache_compact(s.c, 1, s.arr(np.int32([1])), s.arr(np.int32([0])), s.arr(np.int32([0, t])), t, idx.value, t,
                               vals, kc.Betas(beta.value, H * t, t), s.status.value, s.ws.value, s.size, None))
    s.done(1)
    ii = idx.download(np.int32, L * t).reshape(L, t)
    bb = beta.download(np.float32, L * H * t).reshape(L, H, t)
    _, _, kd, vd, b = s.read(1, t)
    for l in range(L):
        assert np.array_equal(kd[l], k[l][ii[l]]), "kept keys"
    assert np.array_equal(b, bb), "beta"
    want_v = (cv.download(np.float32, L * H * t * d).reshape(L, H, t, d).transpose(0, 2, 1, 3) if typ == F32 else
              decode(vo.download(np.uint8, L * t * s.rb).reshape(L, t, -1), typ).reshape(L, t, H, d))
    assert np.array_equal(vd, want_v), "refitted values"
    # two samples share it; each drafts a tree, in its own copy of the last page
    s.ok(dll.kvc_cache_fork(s.c, 2, s.arr(np.int32([1, 1])), s.arr(np.int32([0, 3])), s.status.value, None))
    s.done(2)
    news = [5, 3]
    s.extend([0, 3], news)
    masks = np.uint64([0b1, 0b11, 0b101, 0b1011, 0b10001, 0b1, 0b11, 0b111])
    nk, nv = (rng.standard_normal((L, 8, H, d)).astype(np.float32) for _ in range(2))
    nk, nv = (decode(encode(x.reshape(L, 8, -1), typ), typ).reshape(L, 8, H, d) for x in (nk, nv))
    nq = rng.standard_normal((L, 8, H * G, d))
    for l in range(L):
        s.write(l, [0, 3], news, nk[l], nv[l])
        o, lse, qd = s.attend(l, nq[l], typ, [0, 3], news, masks)
        at = 0
        for n in news:
            rows = slice(at, at + n)
            seen = np.ones((n, t + n), bool)
            seen[:, t:] = [[int(masks[at + i]) >> j & 1 for j in range(n)] for i in range(n)]
            want = attend(qd[rows], np.concatenate([kd[l], nk[l][rows]]), np.concatenate([vd[l], nv[l][rows]]), seen,
                          np.concatenate([bb[l], np.zeros((H, n))], 1), d ** -0.5, typ)
            compare(o[rows], lse[rows].astype(float), want, typ, f"drafts of layer {l}")
            at += n
    # drafts 0, 1 and 3 of the first sample are accepted
    s.ok(dll.kvc_cache_compact(s.c, 1, s.arr(np.int32([0])), s.arr(np.int32([t])), s.arr(np.int32([0, 3])), 3,
                               s.arr(np.int32([0, 1, 3])), 0, None, None, s.status.value, s.ws.value, s.size, None))
    s.done(1)
    _, _, k0, v0, b0 = s.read(0, t + 3)
    assert np.array_equal(k0[:, t:], nk[:, [0, 1, 3]]) and np.array_equal(v0[:, t:], nv[:, [0, 1, 3]])
    assert np.array_equal(k0[:, :t], kd) and np.array_equal(v0[:, :t], vd) and not b0[:, :, t:].any()
    # the shared pages are as they were
    _, _, k1, v1, b1 = s.read(1, t)
    assert np.array_equal(k1, kd) and np.array_equal(v1, vd) and np.array_equal(b1, bb)


def _graph_api():
    import hiprt
    h = hiprt.hip()
    vp = ctypes.c_void_p
    h.hipStreamBeginCapture.argtypes = [vp, ctypes.c_int]
    h.hipStreamEndCapture.argtypes = [vp, ctypes.POINTER(vp)]
    h.hipGraphInstantiate.argtypes = [ctypes.POINTER(vp), vp, vp, vp, ctypes.c_size_t]
    h.hipGraphLaunch.argtypes = [vp, vp]
    h.hipGraphExecDestroy.argtypes = [vp]
    h.hipGraphDestroy.argtypes = [vp]
    return h


def test_captured_steps(lib):
    """A decode step (reserve, write, attend, cut back) in a graph, replayed with other rows and queries between eager
    calls: every replay is the eager result."""
    import hiprt
    dll, h = lib.dll, _graph_api()
    H, G, d, page = 2, 2, 64, 16
    rng = np.random.default_rng(3)
    s = Server(dll, 1, 40, page, 2, 20, H, d, F16, bias=False)
    s.extend([0, 1], [200, 37])
    s.write(0, [0, 1], [200, 37], *(rng.standard_normal((237, H, d)) for _ in range(2)))
    s.ok(dll.kvc_cache_fork(s.c, 1, s.arr(np.int32([1])), s.arr(np.int32([1])), s.status.value, None))   # (refused: itself)
    assert s.status.download(np.int32, 1)[0] == kc.REQ_BAD
    news, n = [3, 2], 5
    rows = [dev(np.zeros(n * s.rb, np.uint8)) for _ in range(2)]
    q = dev(np.zeros((n, H * G, d), np.float16))
    o = dev(np.zeros((n, H * G, d), np.float16))
    lse = dev(np.zeros((n, H * G), np.float32))
    seqs, cu, count, start, zero = (s.arr(np.int32(x)) for x in ([0, 1], [0, 3, 5], news, [200, 37], [0, 0, 0]))
    a = kc.CacheAttnArgs(q=kc.Heads(q.value, H * G * d, d), o=kc.Heads(o.value, H * G * d, d), lse=lse.value, seqs=seqs, cu=cu,
                         n_seq=2, n_tok=n, n_head=H * G, max_new=3, max_len=4096, type=F16)
    size = dll.kvc_attn_cache_workspace(s.c, a)
    assert size > 0     # (a call of two kernels)
    ws = dev(np.zeros(size, np.uint8))

    def step(st):
        s.ok(dll.kvc_cache_extend(s.c, 2, seqs, count, s.status.value, s.ws.value, s.size, st))
        r = [kc.Rows(x.value, 0, s.rb) for x in rows]
        s.ok(dll.kvc_cache_write(s.c, 0, 1, 2, seqs, cu, n, F16, r[0], r[1], st))
        s.ok(dll.kvc_attn_cache(s.c, a, ws.value, size, st))
        s.ok(dll.kvc_cache_compact(s.c, 2, seqs, start, zero, 0, None, 0, None, None, s.status.value, s.ws.value, s.size, st))

    def result(i, run):
        r = np.random.default_rng(100 + i)
        for x in rows:
            x.upload(encode(r.standard_normal((n, H * d)), F16))
        q.upload(r.standard_normal((n, H * G, d)).astype(np.float16))
        run()
        hiprt.synchronize()
        return o.download(np.uint16, n * H * G * d), lse.download(np.uint32, n * H * G), s.len.download(np.int32, 2)

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
        assert want[2].tolist() == [200, 37]
    hiprt.check(h.hipGraphExecDestroy(exe))
    hiprt.check(h.hipGraphDestroy(graph))
    hiprt.check(h.hipStreamDestroy(stream))


def test_two_calls_at_once(lib):
    """Attention of two layers on two streams, each with a workspace of its own, while a third prompt runs."""
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
    cu = s.arr(np.int32([0, 1, 2, 3, 4]))
    calls, streams = [], []
    for l in range(2):
        q = dev(bf16(rng.standard_normal((4, H * G, d))))
        o = dev(np.zeros((4, H * G, d), np.uint16))
        a = kc.CacheAttnArgs(q=kc.Heads(q.value, H * G * d, d), o=kc.Heads(o.value, H * G * d, d), cu=cu, layer=l, type=BF16,
                             n_seq=4, n_tok=4, n_head=H * G, max_new=1, max_len=2000)
        size = dll.kvc_attn_cache_workspace(s.c, a)
        ws = dev(np.zeros(max(size, 16), np.uint8))
        st = ctypes.c_void_p()
        hiprt.check(h.hipStreamCreate(ctypes.byref(st)))
        calls.append((a, q, o, ws, size))
        streams.append(st)

    def one(i, st):
        a, _, _, ws, size = calls[i]
        s.ok(dll.kvc_attn_cache(s.c, a, ws.value, size, st))
    alone = []
    for i in range(2):
        one(i, None)
        hiprt.synchronize()
        alone.append(calls[i][2].download(np.uint16, 4 * H * G * d))
        calls[i][2].zero()
    hiprt.synchronize()
    for _ in range(20):
        for i in range(2):
            one(i, streams[i])
    hiprt.synchronize()
    for i in range(2):
        assert np.array_equal(alone[i], calls[i][2].download(np.uint16, 4 * H * G * d))
        hiprt.check(h.hipStreamDestroy(streams[i]))
    assert not np.array_equal(alone[0], alone[1])


def test_offsets_past_32_bits(lib):
    """The last layer of a cache of more than 4 GiB, and the last pages of it."""
    import hiprt
    dll = lib.dll
    H, G, d, page, pages = 8, 1, 128, 1024, 1100
    if hiprt.mem_free() < 16 << 30:
        pytest.skip("not enough device memory")
    L, rb = 2, 2 * H * d
    K, V = (hiprt.DevBuf(L * pages * page * rb) for _ in range(2))
    assert K.nbytes > 1 << 32
    K.zero()
    V.zero()
    last = [pages - 1, pages - 2]
    rng = np.random.default_rng(1)
    k, v = (bf16(rng.standard_normal((2 * page, H, d))) for _ in range(2))
    for i, p in enumerate(last):
        at = ((L - 1) * pages + p) * page * rb
        K.upload(k[i * page:(i + 1) * page], at)
        V.upload(v[i * page:(i + 1) * page], at)
    refs = np.zeros(pages, np.int32)
    refs[last] = 1
    table, length, drefs = dev(np.int32([last])), dev(np.int32([2 * page])), dev(refs)
    c = kc.KvCache(n_layers=L, n_pages=pages, page_size=page, max_seqs=1, max_pages=2, n_head_kv=H, d_k=d, d_v=d, k_type=BF16,
                   v_type=BF16, K=K.value, V=V.value, table=table.value, len=length.value, refs=drefs.value)
    for new in (1, 40):   # both forms
        q = Strided(rng.standard_normal((new, H, d)), BF16)
        o = Strided(np.zeros((new, H, d)), BF16)
        lse, cu = dev(np.zeros((new, H), np.float32)), dev(np.int32([0, new]))
        a = kc.CacheAttnArgs(q=q.heads(), o=o.heads(), lse=lse.value, cu=cu.value, layer=L - 1, type=BF16, n_seq=1, n_tok=new,
                             n_head=H, max_new=new, max_len=2 * page)
        size = dll.kvc_attn_cache_workspace(c, a)
        ws = dev(np.zeros(max(size, 16), np.uint8))
        assert dll.kvc_attn_cache(c, a, ws.value, size, None) == 0
        seen = np.ones((new, 2 * page), bool)
        seen[:, 2 * page - new:] = np.tril(np.ones((new, new), bool))
        f = lambda x: decode(x.view(np.uint8).reshape(2 * page, -1), BF16).reshape(2 * page, H, d)  # noqa: E731
        want = attend(wide(q._view(q.host), BF16), f(k), f(v), seen, None, d ** -0.5, BF16)
        compare(o.read()[0], lse.download(np.float32, new * H).reshape(new, H).astype(float), want, BF16, f"{new} new")
    # and the rows of that page, read back and moved
    out = dev(np.zeros(L * 5 * rb, np.uint8))
    assert dll.kvc_cache_read(c, 0, page - 2, 5, out.value, None, None, None) == 0
    got = out.download(np.uint16, L * 5 * H * d).reshape(L, 5, H, d)
    assert np.array_equal(got[1], k[page - 2:page + 3]) and not got[0].any()
    size = dll.kvc_cache_workspace(c, 1)
    ws, st = dev(np.zeros(size, np.uint8)), dev(np.zeros(1, np.int32))
    z, cu, idx = dev(np.int32([0])), dev(np.int32([0, 3])), dev(np.int32([7, page + 1, 2 * page - 1]))
    assert dll.kvc_cache_compact(c, 1, z.value, z.value, cu.value, 3, idx.value, 0, None, None, st.value, ws.value, size, None) == 0
    assert dll.kvc_cache_read(c, 0, 0, 3, out.value, None, None, None) == 0
    got = out.download(np.uint16, L * 3 * H * d).reshape(L, 3, H, d)
    assert np.array_equal(got[1], k[[7, page + 1, 2 * page - 1]])
    assert st.download(np.int32, 1)[0] == 0 and drefs.download(np.int32, pages)[last].tolist() == [1, 0]
