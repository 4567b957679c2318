"""Argument checks of include/kvc-cache.h, on a machine without a GPU: every
refusal comes before the device is looked for, and a call that passes the
checks reports KV_COMPACT_E_DEVICE there."""
from __future__ import annotations

import ctypes

import pytest

import kvcompact as kc

FAKE = 1 << 20   # an aligned address that is never read
F32, F16, BF16, Q8_0 = kc.KV_TYPE_F32, kc.KV_TYPE_F16, kc.KV_TYPE_BF16, kc.KV_TYPE_Q8_0


@pytest.fixture(scope="module")
def dll():
    if not kc.product_lib_path().exists():
        pytest.skip("library not built")
    lib = kc.load_product()
    if lib.dll.kv_compact_hip_available():
        pytest.skip("a GPU is there: the calls that pass the checks would run")
    return kc.bind_cache(lib.dll)


def cache(**kw):
    d = dict(n_layers=2, n_pages=8, page_size=16, max_seqs=4, max_pages=4, n_head_kv=2, d_k=64, d_v=64, k_type=F16,
             v_type=F16, K=FAKE, V=FAKE, bias=FAKE, table=FAKE, len=FAKE, refs=FAKE)
    d.update(kw)
    return kc.KvCache(**d)


BAD_CACHES = [
    (dict(K=None), -1), (dict(V=None), -1), (dict(table=None), -1), (dict(len=None), -1), (dict(refs=None), -1),
    (dict(n_layers=0), -2), (dict(n_pages=-1), -2), (dict(max_seqs=0), -2), (dict(max_pages=0), -2),
    (dict(n_head_kv=0), -2), (dict(d_k=0), -2), (dict(d_v=-4), -2),
    (dict(page_size=8), -5), (dict(page_size=48), -5), (dict(page_size=2048), -5), (dict(page_size=0), -5),
    (dict(n_pages=(1 << 20) + 1), -5), (dict(max_pages=(1 << 20) + 1), -5), (dict(d_k=257), -5), (dict(d_v=300), -5),
    (dict(k_type=2), -5), (dict(v_type=3), -5), (dict(k_type=99), -5), (dict(k_type=Q8_0, d_k=48), -5),
    (dict(v_type=Q8_0, d_v=16), -5), (dict(K=FAKE + 8), -5), (dict(V=FAKE + 2), -5), (dict(bias=FAKE + 4), -5), (dict(n_layers=20000), -5),
]


def calls(dll, c):
    """Every cache call with arguments that are right by themselves."""
    size = 1 << 30
    rows = kc.Rows(FAKE, 1 << 16, 256)
    yield dll.kvc_cache_reset(c, None)
    yield dll.kvc_cache_extend(c, 2, FAKE, FAKE, FAKE, FAKE, size, None)
    yield dll.kvc_cache_write(c, 0, 1, 2, FAKE, FAKE, 4, F16, rows, rows, None)
    yield dll.kvc_cache_fork(c, 2, FAKE, FAKE, FAKE, None)
    yield dll.kvc_cache_free(c, 2, FAKE, None)
    yield dll.kvc_cache_compact(c, 2, FAKE, FAKE, FAKE, 4, FAKE, 4, None, None, FAKE, FAKE, size, None)
    yield dll.kvc_cache_read(c, 1, 0, 5, FAKE, FAKE, FAKE, None)
    a = attn()
    yield dll.kvc_attn_cache(c, a, FAKE, size, None)


def attn(**kw):
    h = kc.Heads(FAKE, 4 * 64, 64)
    d = dict(q=h, o=h, lse=None, seqs=None, cu=FAKE, mask=None, mask_words=0, layer=0, type=F16, n_seq=2, n_tok=4, n_head=4,
             max_new=2, max_len=64)
    d.update(kw)
    return kc.CacheAttnArgs(**d)


def test_without_a_gpu(dll):
    assert all(rc == kc.E_DEVICE for rc in calls(dll, cache()))


@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_bad_caches(dll, change, code):
    c = cache(**change)
    assert [rc for rc in calls(dll, c)] == [code] * 8
    assert dll.kvc_cache_workspace(c, 4) == 0 and dll.kvc_attn_cache_workspace(c, attn()) == 0


def test_null_structs(dll):
    assert [rc for rc in calls(dll, None)] == [-1] * 8
    assert dll.kvc_attn_cache(cache(), None, None, 0, None) == -1
    assert dll.kvc_attn_prompt(None, None) == -1


def test_requests(dll):
    c, size = cache(), 1 << 30
    need = dll.kvc_cache_workspace(c, 3)
    assert need > 0 and dll.kvc_cache_workspace(c, 0) == 0 and dll.kvc_cache_workspace(c, 1025) == 0
    for n, code in ((-1, -2), (kc.CACHE_MAX_REQUESTS + 1, -5), (0, 0)):
        assert dll.kvc_cache_extend(c, n, FAKE, FAKE, FAKE, FAKE, size, None) == code
        assert dll.kvc_cache_fork(c, n, FAKE, FAKE, FAKE, None) == code
        assert dll.kvc_cache_free(c, n, FAKE, None) == code
        assert dll.kvc_cache_compact(c, n, FAKE, FAKE, FAKE, 1, FAKE, 1, None, None, FAKE, FAKE, size, None) == code
        assert dll.kvc_cache_write(c, 0, 1, n, FAKE, FAKE, 1, F16, kc.Rows(FAKE, 0, 256), kc.Rows(FAKE, 0, 256), None) == code
    assert dll.kvc_cache_extend(c, 3, FAKE, FAKE, FAKE, FAKE, need - 1, None) == kc.E_SCRATCH
    assert dll.kvc_cache_compact(c, 3, FAKE, FAKE, FAKE, 0, None, 0, None, None, FAKE, FAKE, need - 1, None) == kc.E_SCRATCH
    for k in range(4):
        p = [FAKE] * 4
        p[k] = None
        assert dll.kvc_cache_extend(c, 3, *p, size, None) == -1
    for k in range(3):
        p = [FAKE] * 3
        p[k] = None
        assert dll.kvc_cache_fork(c, 3, *p, None) == -1
    assert dll.kvc_cache_free(c, 3, None, None) == -1


def test_compaction_arguments(dll):
    c, size = cache(), 1 << 30

    def call(c=c, n_idx=4, idx=FAKE, ld=4, v=None, b=None, seqs=FAKE, start=FAKE, cu=FAKE, status=FAKE, ws=FAKE):
        return dll.kvc_cache_compact(c, 2, seqs, start, cu, n_idx, idx, ld, v, b, status, ws, size, None)
    assert call() == kc.E_DEVICE and call(n_idx=0, idx=None) == kc.E_DEVICE
    for name in ("idx", "seqs", "start", "cu", "status", "ws"):
        assert call(**{name: None}) == -1
    assert call(n_idx=-1) == -2 and call(ld=-1) == -2
    assert call(v=kc.Values(None, 0, 0, 0)) == -1 and call(b=kc.Betas(None, 0, 0)) == -1
    assert call(v=kc.Values(FAKE + 1, 0, 256, 128)) == -5 and call(v=kc.Values(FAKE, 0, 255, 128)) == -5
    assert call(v=kc.Values(FAKE, 0, 256, 128)) == kc.E_DEVICE
    assert call(c=cache(k_type=F32, v_type=F32), v=kc.Values(FAKE + 2, 0, 512, 256)) == -5
    assert call(c=cache(bias=None), b=kc.Betas(FAKE, 0, 0)) == -5


def test_write_and_read_arguments(dll):
    c = cache()
    r = kc.Rows(FAKE, 1 << 16, 256)

    def write(c=c, layer=0, n_layers=1, n_rows=4, typ=F16, K=r, V=r, seqs=FAKE, cu=FAKE):
        return dll.kvc_cache_write(c, layer, n_layers, 2, seqs, cu, n_rows, typ, K, V, None)
    for kw, code in ((dict(layer=-1), -2), (dict(layer=2), -2), (dict(layer=1, n_layers=2), -2), (dict(n_layers=-1), -2),
                     (dict(n_rows=-1), -2), (dict(n_layers=0), 0), (dict(n_rows=0), 0), (dict(seqs=None), -1),
                     (dict(cu=None), -1), (dict(K=None), -1), (dict(V=None), -1), (dict(K=kc.Rows(None, 0, 0)), -1),
                     (dict(typ=F32), -5), (dict(typ=BF16), -5), (dict(typ=Q8_0), -5), (dict(typ=7), -5),
                     (dict(K=kc.Rows(FAKE + 1, 0, 256)), -5), (dict(V=kc.Rows(FAKE, 0, 255)), -5),
                     (dict(layer=1), kc.E_DEVICE)):
        assert write(**kw) == code, kw
    q8 = cache(k_type=Q8_0, v_type=Q8_0)
    for typ, code in ((F32, kc.E_DEVICE), (F16, kc.E_DEVICE), (BF16, kc.E_DEVICE), (Q8_0, kc.E_DEVICE), (2, -5)):
        assert write(c=q8, typ=typ) == code
    assert write(c=q8, typ=F32, K=kc.Rows(FAKE + 2, 0, 512)) == -5
    assert write(c=cache(k_type=F32)) == -5
    for args, code in (((-1, 0, 5), -2), ((4, 0, 5), -2), ((0, -1, 5), -2), ((0, 0, -1), -2), ((0, 0, 0), 0)):
        assert dll.kvc_cache_read(c, *args, FAKE, FAKE, FAKE, None) == code
    assert dll.kvc_cache_read(c, 0, 0, 5, None, None, None, None) == 0
    assert dll.kvc_cache_read(c, 0, 0, 5, FAKE + 1, FAKE, FAKE, None) == -5
    assert dll.kvc_cache_read(cache(bias=None), 0, 0, 5, FAKE, FAKE, FAKE, None) == -5


def test_cache_attention_arguments(dll):
    c, h = cache(), kc.Heads(FAKE, 256, 64)

    def call(c=c, ws=FAKE, size=1 << 30, **kw):
        return dll.kvc_attn_cache(c, attn(**kw), ws, size, None)
    none, odd = kc.Heads(None, 256, 64), kc.Heads(FAKE + 1, 256, 64)
    for kw, code in ((dict(), kc.E_DEVICE), (dict(q=none), -1), (dict(o=none), -1), (dict(cu=None), -1),
                     (dict(n_seq=-1), -2), (dict(n_tok=-1), -2), (dict(n_head=0), -2), (dict(n_head=3), -2),
                     (dict(max_new=-1), -2), (dict(max_len=-1), -2), (dict(mask_words=-1), -2), (dict(layer=2), -2),
                     (dict(layer=-1), -2), (dict(n_seq=0), 0), (dict(n_tok=0), 0), (dict(type=F32), -5),
                     (dict(type=BF16), -5), (dict(type=Q8_0), -5), (dict(q=odd), -5), (dict(o=odd), -5)):
        assert call(**kw) == code, kw
    q8 = cache(k_type=Q8_0, v_type=Q8_0)
    for typ, code in ((F16, kc.E_DEVICE), (BF16, kc.E_DEVICE), (F32, -5), (Q8_0, -5)):
        assert call(c=q8, type=typ) == code
    assert call(c=cache(k_type=F16, v_type=BF16)) == -5
    long = dict(n_seq=1, n_tok=1, max_new=1, max_len=100000)
    need = dll.kvc_attn_cache_workspace(c, attn(**long))
    assert need > 0
    assert call(ws=None, **long) == -1 and call(size=need - 1, **long) == kc.E_SCRATCH
    assert call(size=need, **long) == kc.E_DEVICE


def test_prompt_arguments(dll):
    h = kc.Heads(FAKE, 256, 64)
    none, odd = kc.Heads(None, 256, 64), kc.Heads(FAKE + 1, 256, 64)

    def call(**kw):
        d = dict(q=h, k=h, v=h, o=h, lse=None, cu=FAKE, type=F16, n_seq=2, n_tok=9, n_head=4, n_head_kv=2, d_k=64, d_v=64)
        d.update(kw)
        return dll.kvc_attn_prompt(kc.PromptArgs(**d), None)
    for kw, code in ((dict(), kc.E_DEVICE), (dict(q=none), -1), (dict(k=none), -1), (dict(v=none), -1), (dict(o=none), -1),
                     (dict(cu=None), -1), (dict(n_seq=-1), -2), (dict(n_tok=-1), -2), (dict(n_head=0), -2),
                     (dict(n_head_kv=0), -2), (dict(n_head=5), -2), (dict(d_k=0), -2), (dict(d_v=0), -2),
                     (dict(d_k=257), -5), (dict(d_v=512), -5), (dict(type=Q8_0), -5), (dict(type=3), -5), (dict(q=odd), -5),
                     (dict(k=odd), -5), (dict(v=odd), -5), (dict(k=kc.Heads(FAKE, 1 << 23, 64)), -5),
                     (dict(v=kc.Heads(FAKE, -256, 64)), -5), (dict(o=odd), -5), (dict(n_seq=0), 0), (dict(n_tok=0), 0),
                     (dict(type=F32), kc.E_DEVICE), (dict(type=BF16), kc.E_DEVICE)):
        assert call(**kw) == code, kw


def test_struct_sizes():
    # include/kvc-cache.h on x86-64
    assert [ctypes.sizeof(x) for x in (kc.KvCache, kc.Rows, kc.Values, kc.Betas, kc.Heads, kc.PromptArgs,
                                       kc.CacheAttnArgs)] == [88, 24, 32, 24, 24, 144, 120]


def test_sizes_at_the_ends(dll):
    # nothing to do needs no workspace, and rows, cells and blocks stay within what the kernels count with
    c, top, h = cache(), (1 << 31) - 1, kc.Heads(FAKE, 256, 64)
    for kw in (dict(n_seq=0), dict(n_tok=0), dict(n_seq=0, n_tok=0, max_new=0, max_len=0)):
        assert dll.kvc_attn_cache_workspace(c, attn(**kw)) == 0
        assert dll.kvc_attn_cache(c, attn(**kw), None, 0, None) == 0
    size = 1 << 62
    for kw, code in ((dict(n_tok=top), -5), (dict(n_tok=(1 << 28) + 1), -5), (dict(max_new=top), -5),
                     (dict(n_tok=1 << 28), kc.E_DEVICE), (dict(max_len=top), kc.E_DEVICE), (dict(n_seq=top), -5)):
        assert dll.kvc_attn_cache(c, attn(**kw), FAKE, size, None) == code, kw
    for kw, code in ((dict(n_tok=top), -5), (dict(n_tok=(1 << 28) + 1), -5), (dict(n_seq=top), -5),
                     (dict(n_tok=1 << 22), kc.E_DEVICE)):
        d = dict(q=h, k=h, v=h, o=h, lse=None, cu=FAKE, type=F16, n_seq=2, n_tok=9, n_head=4, n_head_kv=2, d_k=64, d_v=64)
        d.update(kw)
        assert dll.kvc_attn_prompt(kc.PromptArgs(**d), None) == code, kw
    r = kc.Rows(FAKE, 0, 256)
    for n, code in ((top, -5), ((1 << 24) + 1, -5), (1 << 24, kc.E_DEVICE)):
        assert dll.kvc_cache_write(c, 0, 1, 2, FAKE, FAKE, n, F16, r, r, None) == code
        assert dll.kvc_cache_read(c, 0, 0, n, FAKE, FAKE, FAKE, None) == code
