"""kvc_cache_weigh (include/kvc-cache.h) where scores are large: their size costs a weight one rounding, in fp32, of a number
of that size, whichever kernel a call takes."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from budget_model import PagedCells
from cache_model import BF16, F16, F32
from kvc_harness import kc
from test_gpu_cache_attn import Strided, dev, dll   # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu

A, B, D, N, CELLS = 35, 25, 64, 256, 300   # every product of a query and a key is 56000, exactly


def scale_of(seed):
    """Scales under which scores are 5000 to 5600, whose products with log2 e are rounded by nearly half a step, up and
    down. (Scores, and scores times log2 e, 7200 to 8100, lie between 2^12 and 2^13, where half a step of fp32 is 2^-12.)"""
    rng = np.random.default_rng(seed)
    s = rng.uniform(5000 / (A * B * D), 5600 / (A * B * D), 4096).astype(np.float32)
    off = (s * np.float32(np.log2(np.e))).astype(np.float64) / (s.astype(np.float64) * np.log2(np.e)) - 1
    return float(s[np.argmax(off)]), float(s[np.argmin(off)])


@pytest.mark.parametrize("typ", [F16, BF16, F32])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("news", [1, 20, N])
@pytest.mark.parametrize("seed", [0, 1])
def test_equal_scores(dll, typ, bias, news, seed):   # noqa: F811
    def edit(k, v, b, cell):
        k[:] = B
        if b is not None:
            b[:] = 0.0
    for scale in scale_of(seed):
        p = PagedCells(typ, [CELLS], 1, D, D, 16, bias, 0, edit=edit)
        q = Strided(np.full((news, 2, D), float(A)), typ)
        score = float(A * B * D) * scale
        lse = np.full((news, 2), score, np.float32)
        lse[1::2] += np.float32(0.25)
        room = p.m.max_pages * 16
        w = dev(np.zeros((p.layer + 1, 3, 1, room), np.float32))
        hold = [dev(np.int32(p.place)), dev(np.int32([0, news])), dev(lse)]
        a = kc.CacheAttnArgs(q=q.heads(), lse=hold[2].value, seqs=hold[0].value, cu=hold[1].value, mask=None, mask_words=0, layer=p.layer,
                             type=typ, n_seq=1, n_tok=news, n_head=2, max_new=news, max_len=CELLS, scale=scale)
        print(f"large scores type={typ} bias={bias} news={news} scale={scale!r}", flush=True)
        assert dll.kvc_cache_weigh(p.ref(), ctypes.byref(a), None, kc.WeighArgs(w.value, 0.0, 0, 0), None) == 0
        got = w.download(np.float32, 3 * (p.layer + 1) * room).reshape(p.layer + 1, 3, room)[p.layer, p.place[0], :CELLS]
        # A row's exponent is off by one rounding of a number of the score's size, and by what goes with the difference, which
        # is under 1: 4 e. Rounded is the score, half a step 2^-12, or the log-sum-exp times log2 e, half a step 2^-12 in
        # powers of two, which is 2^-12 log 2, less. The weight is off by as much relative and 4 e, a sum of R rows by R e.
        e = 2.0 ** -24
        each = np.exp(np.float64(score) - lse.astype(np.float64)).sum(1)
        sees = np.array([each[max(0, j - (CELLS - news)):].sum() for j in range(CELLS)])
        off = np.abs(got - sees) / sees
        assert off.max() <= 1.001 * 2.0 ** -12 + (8 + 2 * news) * e, (off.max(), off.max() * 2.0 ** 12)
