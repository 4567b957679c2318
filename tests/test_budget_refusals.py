"""Argument checks of windows and of a cache's budget (include/kvc-cache.h) on a machine without a GPU: what is refused
before the device is looked for, and what is not (KV_COMPACT_E_DEVICE)."""
from __future__ import annotations

import pytest

import kvcompact as kc
from test_cache_refusals import BAD_CACHES, BF16, F16, F32, FAKE, Q8_0, attn, cache, dll   # noqa: F401 (the fixture)

SIZE = 1 << 40
W = kc.Window(4, 64)


def prompt(**kw):
    h = kc.Heads(FAKE, 256, 64)
    d = dict(q=h, k=h, v=h, o=h, lse=None, cu=FAKE, type=F16, n_seq=2, n_tok=4, n_head=4, n_head_kv=2, d_k=64, d_v=64)
    d.update(kw)
    return kc.PromptArgs(**d)


def pick(**kw):
    d = dict(seqs=FAKE, start=FAKE, keep=FAKE, weight=FAKE, idx=FAKE, ld_idx=8, cu=FAKE, granted=FAKE, status=FAKE, n_idx=8,
             recent=2, heads=kc.HEADS_SUM, max_len=64)
    d.update(kw)
    return kc.PickArgs(**d)


def weigh(**kw):
    d = dict(weight=FAKE, decay=1.0, tail=0, fresh=0)
    d.update(kw)
    return kc.WeighArgs(**d)


def calls(dll, c):   # noqa: F811
    yield dll.kvc_attn_cache_window(c, attn(), W, FAKE, SIZE, None)
    yield dll.kvc_cache_weigh(c, attn(lse=FAKE), W, weigh(), None)
    yield dll.kvc_cache_weigh(c, attn(lse=FAKE), None, weigh(), None)
    yield dll.kvc_cache_pick(c, 2, pick(), FAKE, SIZE, None)
    yield dll.kvc_cache_take_weights(c, 2, FAKE, FAKE, FAKE, FAKE, 4, FAKE, 4, FAKE, FAKE, None)
    yield dll.kvc_cache_take_weights(c, 2, FAKE, FAKE, None, None, 0, None, 0, None, FAKE, None)


def test_without_a_gpu(dll):   # noqa: F811
    assert [rc for rc in calls(dll, cache())] == [kc.E_DEVICE] * 6
    assert dll.kvc_attn_prompt_window(prompt(), W, None) == kc.E_DEVICE


@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_bad_caches(dll, change, code):   # noqa: F811
    c = cache(**change)
    assert [rc for rc in calls(dll, c)] == [code] * 6
    assert dll.kvc_cache_pick_workspace(c, 2, pick()) == 0 and dll.kvc_attn_cache_window_workspace(c, attn(), W) == 0


def test_null_structs(dll):   # noqa: F811
    assert [rc for rc in calls(dll, None)] == [-1] * 6
    c = cache()
    assert dll.kvc_attn_prompt_window(None, W, None) == -1 and dll.kvc_attn_prompt_window(prompt(), None, None) == -1
    assert dll.kvc_attn_cache_window(c, None, W, FAKE, SIZE, None) == -1
    assert dll.kvc_attn_cache_window(c, attn(), None, FAKE, SIZE, None) == -1
    assert dll.kvc_attn_cache_window_workspace(c, attn(max_len=1 << 20), None) == 0
    assert dll.kvc_cache_weigh(c, None, W, weigh(), None) == -1 and dll.kvc_cache_weigh(c, attn(lse=FAKE), W, None, None) == -1
    assert dll.kvc_cache_pick(c, 2, None, FAKE, SIZE, None) == -1 and dll.kvc_cache_pick_workspace(c, 2, None) == 0


@pytest.mark.parametrize("first,last,code", [(0, 1, 0), (-1, 5, -2), (0, 0, -2), (3, -1, -2), ((1 << 31) - 1, (1 << 31) - 1, 0)])
def test_windows(dll, first, last, code):   # noqa: F811
    w, ok = kc.Window(first, last), code or kc.E_DEVICE
    assert dll.kvc_attn_prompt_window(prompt(), w, None) == ok
    assert dll.kvc_attn_cache_window(cache(), attn(), w, FAKE, SIZE, None) == ok
    assert dll.kvc_cache_weigh(cache(), attn(lse=FAKE), w, weigh(), None) == ok
    # (nothing to do is nothing to refuse, but for the window itself)
    assert dll.kvc_attn_prompt_window(prompt(n_tok=0), w, None) == code
    assert dll.kvc_attn_cache_window(cache(), attn(n_seq=0), w, None, 0, None) == code
    assert dll.kvc_cache_weigh(cache(), attn(n_tok=0), w, weigh(weight=None), None) == code


def test_prompt_windows_refuse_what_prompts_do(dll):   # noqa: F811
    h = kc.Heads(FAKE, 256, 64)
    for kw in (dict(n_seq=-1), dict(n_head=3), dict(d_k=0), dict(d_k=257), dict(type=Q8_0), dict(cu=None), dict(n_tok=1 << 29),
               dict(q=kc.Heads(FAKE + 1, 256, 64)), dict(k=kc.Heads(FAKE, 1 << 23, 64)), dict(o=kc.Heads(None, 256, 64)),
               dict(v=h, n_seq=1 << 24), dict(n_seq=0)):
        assert dll.kvc_attn_prompt_window(prompt(**kw), W, None) == dll.kvc_attn_prompt(prompt(**kw), None), kw


def test_cache_windows_refuse_what_attention_does(dll):   # noqa: F811
    for kw in (dict(n_seq=-1), dict(n_head=3), dict(layer=2), dict(max_new=-1), dict(max_len=-1), dict(mask_words=-1), dict(type=BF16),
               dict(n_tok=1 << 29), dict(q=kc.Heads(FAKE + 1, 256, 64)), dict(o=kc.Heads(None, 256, 64)), dict(cu=None),
               dict(n_seq=1 << 23)):
        assert dll.kvc_attn_cache_window(cache(), attn(**kw), W, FAKE, SIZE, None) == dll.kvc_attn_cache(cache(), attn(**kw), FAKE, SIZE, None), kw
    assert dll.kvc_attn_cache_window(cache(v_type=F32), attn(), W, FAKE, SIZE, None) == -5


def test_window_workspace(dll):   # noqa: F811
    # goes with what a token can see, not with what the sequence holds
    c, a = cache(), attn(max_len=1 << 20)
    full, near = dll.kvc_attn_cache_workspace(c, a), dll.kvc_attn_cache_window_workspace(c, a, kc.Window(4, 2000))
    assert full > near > 0 and dll.kvc_attn_cache_window_workspace(c, a, W) == 0
    assert dll.kvc_attn_cache_window_workspace(c, a, kc.Window(1 << 30, 1)) == full
    assert dll.kvc_attn_cache_window(c, a, kc.Window(4, 2000), FAKE, near - 1, None) == kc.E_SCRATCH
    assert dll.kvc_attn_cache_window(c, a, kc.Window(4, 2000), None, near, None) == -1
    assert dll.kvc_attn_cache_window(c, a, kc.Window(4, 2000), FAKE + 4, near, None) == -5
    assert dll.kvc_attn_cache_window(c, a, kc.Window(4, 2000), FAKE, near, None) == kc.E_DEVICE
    assert dll.kvc_attn_cache_window_workspace(c, a, kc.Window(0, 0)) == 0


def test_weighing(dll):   # noqa: F811
    def call(c=cache(), w=W, x=weigh(), **kw):
        return dll.kvc_cache_weigh(c, attn(**{"lse": FAKE, **kw}), w, x, None)
    assert call() == kc.E_DEVICE and call(o=kc.Heads(None, 0, 0)) == kc.E_DEVICE   # (o is not looked at)
    for kw, code in ((dict(lse=None), -1), (dict(cu=None), -1), (dict(q=kc.Heads(None, 256, 64)), -1), (dict(x=weigh(weight=None)), -1),
                     (dict(x=weigh(decay=-0.5)), -2), (dict(x=weigh(decay=1.5)), -2), (dict(x=weigh(decay=float("nan"))), -2),
                     (dict(x=weigh(tail=-1)), -2), (dict(x=weigh(fresh=-1)), -2), (dict(x=weigh(weight=FAKE + 2)), -5),
                     (dict(q=kc.Heads(FAKE + 1, 256, 64)), -5), (dict(type=BF16), -5), (dict(n_head=3), -2), (dict(layer=-1), -2),
                     (dict(n_seq=1 << 23), -5), (dict(c=cache(v_type=F32)), -5), (dict(n_seq=0), 0), (dict(n_tok=0), 0)):
        assert call(**kw) == code, kw


def test_picking(dll):   # noqa: F811
    c = cache()
    need = dll.kvc_cache_pick_workspace(c, 3, pick())
    assert need == 4 * 2 * 3 * 64 and dll.kvc_cache_pick_workspace(c, 3, pick(ld_idx=0)) == need // 2
    # (no sequence is longer than its table's row: 4 pages of 16)
    assert dll.kvc_cache_pick_workspace(c, 3, pick(max_len=1 << 30)) == need
    for n, code in ((-1, -2), (kc.CACHE_MAX_REQUESTS + 1, -5), (0, 0)):
        assert dll.kvc_cache_pick(c, n, pick(), FAKE, SIZE, None) == code
        assert dll.kvc_cache_pick_workspace(c, n, pick()) == 0
    for kw in (dict(seqs=None), dict(start=None), dict(keep=None), dict(weight=None), dict(idx=None), dict(cu=None),
               dict(granted=None), dict(status=None)):
        assert dll.kvc_cache_pick(c, 3, pick(**kw), FAKE, SIZE, None) == -1, kw
    for kw in (dict(n_idx=-1), dict(recent=-1), dict(max_len=-1), dict(ld_idx=-1), dict(ld_idx=7), dict(heads=2), dict(heads=-1)):
        assert dll.kvc_cache_pick(c, 3, pick(**kw), FAKE, SIZE, None) == -2, kw
        assert dll.kvc_cache_pick_workspace(c, 3, pick(**kw)) == 0
    assert dll.kvc_cache_pick(c, 3, pick(weight=FAKE + 4), FAKE, SIZE, None) == -5
    assert dll.kvc_cache_pick(c, 3, pick(), None, SIZE, None) == -1
    assert dll.kvc_cache_pick(c, 3, pick(), FAKE + 4, SIZE, None) == -5
    assert dll.kvc_cache_pick(c, 3, pick(), FAKE, need - 1, None) == kc.E_SCRATCH
    assert dll.kvc_cache_pick(c, 3, pick(n_idx=0, idx=None), FAKE, need, None) == kc.E_DEVICE
    assert dll.kvc_cache_pick(c, 3, pick(max_len=0), None, 0, None) == kc.E_DEVICE
    wide = cache(n_layers=16384, k_type=F32, v_type=F32)
    assert dll.kvc_cache_pick(wide, 256, pick(), FAKE, SIZE, None) == -5
    assert dll.kvc_cache_pick(wide, 255, pick(), FAKE, SIZE, None) == kc.E_DEVICE
    assert dll.kvc_cache_pick(wide, 1024, pick(ld_idx=0), FAKE, SIZE, None) == kc.E_DEVICE


def test_taking(dll):   # noqa: F811
    c = cache()

    def call(n=2, src=FAKE, dst=FAKE, start=FAKE, cu=FAKE, n_idx=4, idx=FAKE, ld=4, status=FAKE, weight=FAKE):
        return dll.kvc_cache_take_weights(c, n, src, dst, start, cu, n_idx, idx, ld, status, weight, None)
    assert call() == kc.E_DEVICE and call(status=None) == kc.E_DEVICE and call(ld=0) == kc.E_DEVICE
    for name in ("src", "dst", "start", "idx", "weight"):
        assert call(**{name: None}) == -1, name
    assert call(n_idx=0, idx=None) == kc.E_DEVICE
    assert call(cu=None, start=None, idx=None) == kc.E_DEVICE   # (whole sequences, after a fork)
    assert call(n_idx=-1) == -2 and call(ld=-1) == -2 and call(weight=FAKE + 2) == -5
    for n, code in ((-1, -2), (kc.CACHE_MAX_REQUESTS + 1, -5), (0, 0)):
        assert call(n=n) == code
