"""kvc_cache_weigh (include/kvc-cache.h) where a block goes on to further tiles of cells: sequences with more cells than the
call says, and enough rows for the kernels that take cells by tiles."""
from __future__ import annotations

import pytest

from cache_model import F32
from test_gpu_cache_attn import KINDS, dll   # noqa: F401 (the fixture)
from test_gpu_weigh import run_weigh

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("said", [1, 32, 300])
@pytest.mark.parametrize("window", [None, (20, 50), (200, 90)])
def test_more_cells_than_said(dll, typ, cache, d, said, window):   # noqa: F811
    run_weigh(dll, typ, cache, [700, 401, 30], [90, 140, 30], 1, 2, d, page=32, window=window, decay=0.5, seed=d + said, max_len=said,
              runs=2)
    run_weigh(dll, typ, cache, [700, 401, 30], [90, 140, 30], 2, 3, d, page=32, window=window, decay=1.0, bias=True, tree=True, words=2,
              seed=d + said, max_len=said, runs=2)


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tail", [35, 65, 100])
def test_last_tokens_of_more_cells_than_said(dll, typ, cache, d, tail):   # noqa: F811
    # (the last tokens see the first cells and a window of cells behind a gap of whole tiles)
    G = 2 if cache == F32 else 4
    run_weigh(dll, typ, cache, [900, 500], [200, 500], 1, G, d, page=16, window=(40, 30), tail=tail, decay=0.5, seed=d, max_len=1, runs=2)
    run_weigh(dll, typ, cache, [900, 500], [200, 500], 1, G, d, page=16, tail=tail, decay=0.0, seed=d, max_len=1, runs=2)


@pytest.mark.parametrize("typ,cache", KINDS)
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 1)])
def test_many_sequences_of_more_cells_than_said(dll, typ, cache, pad, shift):   # noqa: F811
    # (enough of them for blocks that do not share out rows)
    lens = [300 + 7 * i % 200 for i in range(140)]
    run_weigh(dll, typ, cache, lens, [35 + i % 7 for i in range(140)], 4, 4, 64, page=64, window=(10, 40), decay=0.5, seed=3, max_len=128,
              pad=pad, shift=shift, runs=2)
