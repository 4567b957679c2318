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
