"""kvc_cache_weigh (include/kvc-cache.h): a row whose log-sum-exp is -inf gives nothing, whatever its query holds."""
from __future__ import annotations

import numpy as np
import pytest

import test_gpu_weigh
from cache_model import BF16, F16, F32, Q8_0
from test_gpu_cache_attn import KINDS, Strided, dll   # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


def run(dll, monkeypatch, typ, cache, lens, news, G, d, rows, **more):   # noqa: F811
    """Rows (token, head) of each sequence whose queries are not finite, and whose log-sum-exps are -inf."""
    cu = np.concatenate([[0], np.cumsum(news)])

    def queries(x, *a):
        x = x.copy()
        for s, n in enumerate(news):
            for j, (i, h) in enumerate(rows(n)):
                x[cu[s] + i, h, j % 3::2] = (np.nan, np.inf, -np.inf)[j % 3]
        return Strided(x, *a)

    def edit(lse, s):
        for i, h in rows(news[s]):
            lse[i, h] = -np.inf
    monkeypatch.setattr(test_gpu_weigh, "Strided", queries)
    got = test_gpu_weigh.run_weigh(dll, typ, cache, lens, news, 1, G, d, lse_edit=edit, **more)
    assert not np.isnan(got).any()


def some(n):   # some rows, whole tokens among them, and the last one, which fills up a tile
    return [(i, h) for i in range(0, n, 3) for h in (0, 1) if (i + h) % 2 == 0] + [(n - 1, 0), (n - 1, 1)]


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("news", [[1, 1], [8, 3], [20, 15], [60, 40]])
@pytest.mark.parametrize("window", [None, (4, 30)])
def test_few_tokens(dll, monkeypatch, typ, cache, d, news, window):   # noqa: F811
    run(dll, monkeypatch, typ, cache, [150, 70], news, 2, d, some, window=window, decay=0.5, seed=d)
    run(dll, monkeypatch, typ, cache, [150, 70], news, 2, d, some, window=window, decay=0.5, seed=d, tree=True, bias=True)


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("announced", [None, 1 << 20])
@pytest.mark.parametrize("bias", [False, True])
def test_many_tokens(dll, monkeypatch, typ, cache, d, announced, bias):   # noqa: F811
    # (more cells announced: more blocks, of fewer waves)
    run(dll, monkeypatch, typ, cache, [400, 300], [150, 131], 2, d, some, bias=bias, decay=1.0, seed=d, max_len=announced)
    run(dll, monkeypatch, typ, cache, [400, 300], [150, 131], 3, d, some, bias=bias, decay=0.5, seed=d, max_len=announced,
        window=(20, 100))
    run(dll, monkeypatch, typ, cache, [400, 300], [150, 131], 2, d, lambda n: [(n - 1, 1), (n // 2, 0)], bias=bias, tree=True, words=3,
        decay=1.0, seed=d, max_len=announced)


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("d", [20, 72])
@pytest.mark.parametrize("news", [[1, 2], [20, 15], [150, 60]])
def test_odd_heads(dll, monkeypatch, typ, d, news):   # noqa: F811
    run(dll, monkeypatch, typ, typ, [200, 70], news, 2, d, some, pad=1, shift=1, decay=0.5, seed=d)


@pytest.mark.parametrize("typ", [F16, BF16])
def test_every_row(dll, monkeypatch, typ):   # noqa: F811
    for cache in (typ, Q8_0):
        for news in ([1, 1], [30, 20], [150, 60]):
            run(dll, monkeypatch, typ, cache, [200, 70], news, 2, 64, lambda n: [(i, h) for i in range(n) for h in (0, 1)], decay=0.5)
