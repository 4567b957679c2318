"""Arguments of include/kvc-cache.h beyond those of test_cache_refusals.py, on a
machine without a GPU: what is refused, and what is not."""
from __future__ import annotations

import kvcompact as kc
from test_cache_refusals import BF16, F16, F32, FAKE, Q8_0, attn, cache, dll   # noqa: F401 (the fixture)


def test_granted_reservations(dll):   # noqa: F811
    c, size = cache(), 1 << 30
    need = dll.kvc_cache_workspace(c, 3)
    for granted in (FAKE, None):
        assert dll.kvc_cache_extend_granted(c, 3, FAKE, FAKE, FAKE, granted, FAKE, size, None) == kc.E_DEVICE
        assert dll.kvc_cache_extend_granted(c, 3, FAKE, FAKE, FAKE, granted, FAKE, need - 1, None) == kc.E_SCRATCH
        for n, code in ((-1, -2), (kc.CACHE_MAX_REQUESTS + 1, -5), (0, 0)):
            assert dll.kvc_cache_extend_granted(c, n, FAKE, FAKE, FAKE, granted, FAKE, size, None) == code
        for k in range(4):
            p = [FAKE, FAKE, FAKE, granted, FAKE]
            p[k if k < 3 else 4] = None
            assert dll.kvc_cache_extend_granted(c, 3, *p, size, None) == -1
    assert dll.kvc_cache_extend_granted(None, 3, FAKE, FAKE, FAKE, FAKE, FAKE, size, None) == -1


def test_given_values_beside_keys_of_another_type(dll):   # noqa: F811
    # what the V rows are asked for goes by V's type alone, whatever a row of K takes
    for kt, H, dk in ((F16, 1, 33), (BF16, 3, 7), (Q8_0, 1, 32), (F16, 2, 64), (F32, 2, 64)):
        for vt, d_v, step in ((F32, 5, 4), (F16, 5, 2), (Q8_0, 32, 2)):
            c = cache(n_head_kv=H, d_k=dk, d_v=d_v, k_type=kt, v_type=vt)

            def call(v):
                return dll.kvc_cache_compact(c, 2, FAKE, FAKE, FAKE, 4, FAKE, 4, v, None, FAKE, FAKE, 1 << 30, None)
            right = [FAKE + step, 3 * step, 5 * step, 7 * step]
            assert call(kc.Values(*right)) == kc.E_DEVICE
            for i in range(4):
                wrong = list(right)
                wrong[i] += step // 2
                assert call(kc.Values(*wrong)) == -5


def test_caches_of_two_types(dll):   # noqa: F811
    # rows are reserved, shared, moved and read; only same types are written and attended
    c, size, r = cache(k_type=F16, v_type=F32), 1 << 30, kc.Rows(FAKE, 0, 512)
    assert dll.kvc_cache_reset(c, None) == kc.E_DEVICE
    assert dll.kvc_cache_extend(c, 2, FAKE, FAKE, FAKE, FAKE, size, None) == kc.E_DEVICE
    assert dll.kvc_cache_compact(c, 2, FAKE, FAKE, FAKE, 4, FAKE, 4, None, None, FAKE, FAKE, size, None) == kc.E_DEVICE
    assert dll.kvc_cache_read(c, 1, 0, 5, FAKE, FAKE, FAKE, None) == kc.E_DEVICE
    for typ in (F32, F16, BF16, Q8_0):
        assert dll.kvc_cache_write(c, 0, 1, 2, FAKE, FAKE, 4, typ, r, r, None) == -5
        assert dll.kvc_attn_cache(c, attn(type=typ), FAKE, size, None) == -5


def test_workspace_that_is_not_needed(dll):   # noqa: F811
    # any address will do where the call needs no workspace; where it does, 16-byte aligned ones
    c, size = cache(), 1 << 30
    short, long = attn(), attn(n_seq=1, n_tok=1, max_new=1, max_len=100000)
    assert dll.kvc_attn_cache_workspace(c, short) == 0 and dll.kvc_attn_cache_workspace(c, long) > 0
    for ws, code in ((None, -1), (FAKE + 4, -5), (FAKE + 8, -5), (FAKE + 16, kc.E_DEVICE)):
        assert dll.kvc_attn_cache(c, short, ws, size, None) == kc.E_DEVICE
        assert dll.kvc_attn_cache(c, long, ws, size, None) == code


def test_what_one_launch_takes(dll):   # noqa: F811
    # a cache call shapes its launch to what there is: only sequences times KV heads are limited
    c = cache(k_type=F32, v_type=F32, n_head_kv=8)
    for kw, code in ((dict(n_seq=2048, max_new=32768), kc.E_DEVICE), (dict(n_seq=1 << 19, max_new=1 << 19), kc.E_DEVICE),
                     (dict(n_seq=(1 << 20) - 1, max_new=1), kc.E_DEVICE), (dict(n_seq=1 << 20, max_new=1), -5)):
        a = attn(type=F32, n_head=8, max_len=1 << 20, **kw)
        assert dll.kvc_attn_cache_workspace(c, a) == 0 and dll.kvc_attn_cache(c, a, None, 0, None) == code, kw

    # a prompt call: n_head_kv * (ceil(n_tok * n_head / n_head_kv / R) + n_seq) < 2^23
    def prompt(typ, d, n_tok, n_seq=1, pad=0, G=2):
        h = [kc.Heads(FAKE, x * d + pad, d) for x in (2 * G, 2, 2, 2 * G)]
        return dll.kvc_attn_prompt(kc.PromptArgs(q=h[0], k=h[1], v=h[2], o=h[3], cu=FAKE, type=typ, n_seq=n_seq, n_tok=n_tok,
                                                 n_head=2 * G, n_head_kv=2, d_k=d, d_v=d), None)
    for typ, d, pad, R in ((F16, 64, 0, 128), (BF16, 256, 8, 128), (F32, 128, 0, 32), (F32, 256, 0, 16), (F32, 132, 4, 16),
                           (F16, 64, 1, 16), (F16, 20, 0, 16), (F32, 64, 1, 16)):
        for n_seq in (1, 1 << 20):
            most = ((1 << 22) - 1 - n_seq) * R // 2      # tokens: G rows each, R rows a block
            if most * 4 > 1 << 30:
                continue
            assert prompt(typ, d, most, n_seq, pad) == kc.E_DEVICE, (typ, d, pad)
            assert prompt(typ, d, most + 1, n_seq, pad) == -5, (typ, d, pad)
