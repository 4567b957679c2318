"""Launches of the cache's attention at the ends of what they are shaped for
(include/kvc-cache.h)."""
from __future__ import annotations

import pytest

from cache_model import BF16, F16, F32, Q8_0
from test_gpu_cache_attn import dll, run_cells   # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ,cache", [(F32, F32), (BF16, BF16), (F16, Q8_0)])
@pytest.mark.parametrize("d", [64, 128])
def test_more_announced_than_a_launch_holds(dll, typ, cache, d):   # noqa: F811
    # 160 sequences of up to 2^20 new tokens would be more blocks than one launch takes
    lens = [70 + i % 30 if i % 40 == 0 else 3 + i % 5 for i in range(160)]
    news = [40 + i % 20 if i % 40 == 0 else 1 + i % 3 for i in range(160)]
    run_cells(dll, typ, cache, lens, news, 1, 2, d, d, tree=True, seed=40, max_new=1 << 20, max_len=1 << 20)


@pytest.mark.parametrize("typ,cache", [(F32, F32), (BF16, BF16), (F16, Q8_0)])
def test_longest_cache_announced(dll, typ, cache):   # noqa: F811
    for news in ([1, 1], [40, 9]):
        run_cells(dll, typ, cache, [300, 90], news, 1, 2, 64, 64, seed=41, max_len=(1 << 31) - 1, runs=2)
