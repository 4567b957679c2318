"""k_weigh_rows lane by lane on the CPU (tests/waves): what passes between the waves of a block is ordered by block
barriers, whichever wave runs first, also where a block has several tiles of cells and some that no token sees."""
from __future__ import annotations

import re
import shutil
import struct
import subprocess
from pathlib import Path

import numpy as np
import pytest

from budget_model import window_seen
from test_gpu_weigh import log_sums, weights_of

HERE = Path(__file__).resolve().parent
CSRC = HERE.parent / "kv-compact_amd" / "csrc"
CLANG = "/opt/rocm/llvm/bin/clang++"


def cut(name, begin, end):
    m = re.search(rf"^{begin}.*?(?=^{end})", (CSRC / name).read_text(), re.S | re.M)
    assert m, f"{name}: {begin} not found"
    return m.group(0)


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    if not shutil.which(CLANG):
        pytest.skip("clang++ not available")
    d = tmp_path_factory.mktemp("weigh")
    text = (cut("kvc_attn_kernels.h", "// Where rows of K or V stand", "namespace {") +
            cut("kvc_attn_kernels.h", "typedef float f4", "// Tiles of a block's key range") +
            cut("kvc_attn_kernels.h", "// A bf16 row over Q8_0 keys", "template <int TYPE, int QT, int D, int RT, Columns COLS, bool WINDOW>") +
            cut("kvc_weigh.hip", "struct WeighArgs", "// Few rows: 16 RT"))
    text = re.sub(r"asm volatile\(.*?\);", ";", text, flags=re.S).replace("__attribute__((address_space(4)))", "")
    (d / "weigh_rows.inc").write_text(text)
    b = subprocess.run([CLANG, "-std=c++17", "-O1", "-g", "-w", "-mf16c", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                        f"-I{d}", str(HERE / "waves" / "weigh_rows.cpp"), "-o", str(d / "weigh_rows")],
                       capture_output=True, text=True, timeout=300)
    assert b.returncode == 0, b.stderr[-3000:]
    return d / "weigh_rows"


def run(exe, split, first, cells, tokens, window, tiles, H=1, G=4, page=16, decay=0.5, seed=0, out=()):
    rng = np.random.default_rng(seed)
    pages = -(-cells // page)
    n_pages = pages + 1
    table = rng.permutation(n_pages)[:pages].astype(np.int32)
    q = rng.standard_normal((tokens, H * G, 64)).astype(np.float32)
    k = rng.standard_normal((n_pages, page, H, 64)).astype(np.float32)
    old = np.exp(rng.standard_normal((H, pages * page))).astype(np.float32)
    seen = window_seen(cells, tokens, window[0], window[1])
    rows = k[table].reshape(-1, H, 64)[:cells].astype(np.float64)
    lse = log_sums(q.astype(np.float64), rows, None, seen, 0.125)
    for i, h in out:   # rows whose log-sum-exp is -inf, and whose queries are not finite
        lse[i, h] = -np.inf
        q[i, h, i % 5::7] = np.nan if i % 2 else np.inf
    want, tol = weights_of(q.astype(np.float64), rows, None, seen, 0.125, lse.astype(np.float64), 0)
    had = old[:, :cells].astype(np.float64)
    had[:, cells - tokens:] = 0
    head = struct.pack("<11if", split, first, H, G, page, n_pages, cells, tokens, *window, tiles, decay)
    r = subprocess.run([str(exe)], input=head + b"".join(x.tobytes() for x in (table, q, k, lse, old)), capture_output=True, timeout=300)
    assert r.returncode == 0, r.stderr.decode()[-3000:]
    got = np.frombuffer(r.stdout, np.float32).reshape(old.shape)
    off = np.abs(got[:, :cells] - (decay * had + want))
    assert (off <= tol + 2.0 ** -22 * had).all(), np.argwhere(off > tol + 2.0 ** -22 * had)[:5].tolist()
    assert np.array_equal(got[:, cells:], old[:, cells:])


@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("first", [0, 1, 2, 3, -1])
@pytest.mark.parametrize("tiles", [1, 3])
def test_tiles_that_no_token_sees(exe, split, first, tiles):
    # (tiles of 32 cells, or of 128: first cells, hidden ones, the window's; twenty tokens of four heads)
    run(exe, split, first, 400, 20, (20, 30), tiles)


@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("first", [0, 1, -1])
def test_prompts(exe, split, first):
    run(exe, split, first, 150, 150, (0, 1 << 30), 1, H=2, G=3)
    run(exe, split, first, 150, 40, (5, 20), 2, H=2, G=3, page=32)


@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("first", [0, 1, 2, 3, -1])
def test_rows_left_out(exe, split, first):
    # (their scores are NaN: tiles of cells are gone through twice, beside others that no token sees)
    run(exe, split, first, 400, 20, (20, 30), 1, out=[(3, 0), (8, 2), (19, 3)])
    run(exe, split, first, 300, 60, (0, 1 << 30), 1, G=2, out=[(0, 0), (33, 1), (59, 1)])
    run(exe, split, first, 200, 40, (5, 20), 2, G=2, out=[(i, h) for i in range(40) for h in (0, 1)])
