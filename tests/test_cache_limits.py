"""Arguments of include/kvc-cache.h beyond those of test_cache_refusals.py, on a
machine without a GPU: what is refused, and what is not."""
from __future__ import annotations

import kvcompact as kc
from test_cache_refusals import FAKE, cache, dll   # noqa: F401 (the fixture)


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
