"""The cache's calls as they meet in a server (include/kvc-cache.h): prompts and
cells attended at once on streams of their own, and a Q8_0 cache from its
prompt through a compaction to the attention that reads it."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from cache_model import BF16, F16, F32, Q8_0, attend, bf16, decode, encode
from kvc_harness import kc
from test_gpu_cache_attn import Strided, compare, wide
from test_gpu_cache_run import Server, _graph_api, dev, lib   # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


def test_prompts_beside_cells(lib):   # noqa: F811
    """Cells of two layers and a batch of prompts on three streams: every round has queries and results of its own, and
    each result is, bit for bit, what the call gives alone."""
    import hiprt
    dll, h = lib.dll, _graph_api()
    H, G, d, page, n_seq, rounds = 4, 2, 128, 32, 4, 12
    rng = np.random.default_rng(19)
    s = Server(dll, 2, 300, page, n_seq, 70, H, d, BF16, bias=False)
    lens = [2000, 1500, 900, 64]
    s.extend(range(n_seq), lens)
    for l in range(2):
        s.write(l, range(n_seq), lens, *(rng.standard_normal((sum(lens), H, d)) for _ in range(2)))
    cu, pcu = s.arr(np.arange(5, dtype=np.int32)), s.arr(np.int32([0, 700, 733, 1500]))
    pk, pv = (dev(bf16(rng.standard_normal((1500, H, d)))) for _ in range(2))
    calls = []                                  # (entry, structs, o, lse, elements, rows)
    for i in range(rounds):
        for l in range(3):
            n = 1500 if l == 2 else n_seq
            q = dev(bf16(rng.standard_normal((n, H * G, d))))
            o, lse = dev(np.zeros((n, H * G, d), np.uint16)), dev(np.zeros((n, H * G), np.float32))
            hq, ho = kc.Heads(q.value, H * G * d, d), kc.Heads(o.value, H * G * d, d)
            s.keep += [q]
            if l == 2:
                a = kc.PromptArgs(q=hq, k=kc.Heads(pk.value, H * d, d), v=kc.Heads(pv.value, H * d, d), o=ho, lse=lse.value,
                                  cu=pcu, type=BF16, n_seq=3, n_tok=n, n_head=H * G, n_head_kv=H, d_k=d, d_v=d)
            else:
                a = kc.CacheAttnArgs(q=hq, o=ho, lse=lse.value, cu=cu, layer=l, type=BF16, n_seq=n_seq, n_tok=n,
                                     n_head=H * G, max_new=1, max_len=2000)
            calls.append((l, a, o, lse, n * H * G * d, n * H * G))
    size = dll.kvc_attn_cache_workspace(s.c, calls[0][1])
    assert size > 0
    ws = [dev(np.zeros(size, np.uint8)) for _ in range(2)]

    def queue(call, stream):
        l, a = call[:2]
        s.ok(dll.kvc_attn_prompt(a, stream) if l == 2 else dll.kvc_attn_cache(s.c, a, ws[l].value, size, stream))

    def results():
        hiprt.synchronize()
        out = [(o.download(np.uint16, n), lse.download(np.uint32, m)) for _, _, o, lse, n, m in calls]
        for _, _, o, lse, _, _ in calls:
            o.zero()
            lse.zero()
        hiprt.synchronize()
        return out

    for c in calls:
        queue(c, None)
        hiprt.synchronize()
    alone = results()
    streams = [ctypes.c_void_p() for _ in range(3)]
    for st in streams:
        hiprt.check(h.hipStreamCreate(ctypes.byref(st)))
    for _ in range(3):
        for c in calls:
            queue(c, streams[c[0]])
        for i, (a, b) in enumerate(zip(alone, results())):
            assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1]), f"round {i // 3}, call {i % 3}"
    assert len({a[0].tobytes() for a in alone}) == len(alone)
    for st in streams:
        hiprt.check(h.hipStreamDestroy(st))


@pytest.mark.parametrize("typ", [F16, BF16])
def test_q8_0_from_prompt_to_drafts(lib, typ):   # noqa: F811
    """Rows encoded into a Q8_0 cache, compacted there (keys in place, values refitted and encoded, beta fitted), shared
    and drafted on: each attention is the one of what the cache then holds."""
    dll = lib.dll
    L, H, G, d, page, T = 2, 2, 2, 64, 32, 600
    rng = np.random.default_rng(7)
    s = Server(dll, L, 80, page, 4, 40, H, d, Q8_0)
    k, v = (rng.standard_normal((L, T, H, d)).astype(np.float32) for _ in range(2))

    def stored(x):
        return decode(encode(x.reshape(*x.shape[:2], -1), Q8_0), Q8_0).reshape(x.shape)

    s.extend([1], [T])
    for l in range(L):
        rows = [kc.Rows(s.arr(x[l]), 0, 4 * H * d) for x in (k, v)]
        s.ok(dll.kvc_cache_write(s.c, l, 1, 1, s.arr(np.int32([1])), s.arr(np.int32([0, T])), T, F32, *rows, None))
    kb, vb, kd, vd, b = s.read(1, T)
    assert np.array_equal(kd, stored(k)) and np.array_equal(vd, stored(v)) and not b.any()
    p = lib.params(target_ratio=0.2, skip_beta=0, use_cheap_qref=1)
    t, _ = kc.plan(dll, T, 0, False, p)
    idx, beta, cv, st = (dev(np.zeros(n, np.float32)) for n in (L * t, L * H * t, L * H * t * d, L * 3))
    ko, vo = (dev(np.zeros(L * t * s.rb, np.uint8)) for _ in range(2))
    s.ok(dll.kvc_compact_quantized_layers_device(kb.value, vb.value, None, L, Q8_0, Q8_0, s.rb, s.rb, T, 0, H, d, d,
                                                 T * s.rb, T * s.rb, 0, p,
                                                 kc.DeviceOut(idx.value, beta.value, cv.value, st.value), ko.value, vo.value, None))
    # the compacted sequence is one of two that share the prompt
    s.ok(dll.kvc_cache_fork(s.c, 1, s.arr(np.int32([1])), s.arr(np.int32([2])), s.status.value, None))
    s.done(1)
    s.ok(dll.kvc_cache_compact(s.c, 1, s.arr(np.int32([2])), s.arr(np.int32([0])), s.arr(np.int32([0, t])), t, idx.value, t,
                               kc.Values(vo.value, t * s.rb, s.rb, s.rb // H), kc.Betas(beta.value, H * t, t), s.status.value,
                               s.ws.value, s.size, None))
    s.done(1)
    ii = idx.download(np.int32, L * t).reshape(L, t)
    bb = beta.download(np.float32, L * H * t).reshape(L, H, t)
    _, _, k2, v2, b2 = s.read(2, t)
    assert all(np.array_equal(k2[l], kd[l][ii[l]]) for l in range(L)) and np.array_equal(b2, bb)
    assert np.array_equal(v2, decode(vo.download(np.uint8, L * t * s.rb).reshape(L, t, -1), Q8_0).reshape(L, t, H, d))
    # both are drafted on at once, the long one without a bias
    news, masks = [4, 3], np.uint64([0b1, 0b11, 0b101, 0b1101, 0b1, 0b11, 0b101])
    s.extend([2, 1], news)
    nk, nv = (rng.standard_normal((L, 7, H, d)).astype(np.float32) for _ in range(2))
    nq = rng.standard_normal((L, 7, H * G, d))
    for l in range(L):
        rows = [kc.Rows(s.arr(x[l]), 0, 4 * H * d) for x in (nk, nv)]
        s.ok(dll.kvc_cache_write(s.c, l, 1, 2, s.arr(np.int32([2, 1])), s.arr(np.int32([0, 4, 7])), 7, F32, *rows, None))
        o, lse, qd = s.attend(l, nq[l], typ, [2, 1], news, masks)
        at = 0
        for n, (hk, hv, hb) in zip(news, ((k2, v2, bb), (kd, vd, np.zeros((L, H, T))))):
            r, m = slice(at, at + n), hk.shape[1]
            seen = np.ones((n, m + n), bool)
            seen[:, m:] = [[int(masks[at + i]) >> j & 1 for j in range(n)] for i in range(n)]
            want = attend(qd[r], np.concatenate([hk[l], stored(nk)[l][r]]), np.concatenate([hv[l], stored(nv)[l][r]]), seen,
                          np.concatenate([hb[l], np.zeros((H, n))], 1), d ** -0.5, typ)
            compare(o[r], lse[r].astype(float), want, typ, f"drafts of layer {l} over {m} cells")
            at += n
