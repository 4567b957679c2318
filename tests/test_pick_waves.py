"""kvc_cache_pick's kernels lane by lane on the CPU (tests/waves): what passes between the waves of a block is ordered by
block barriers, whichever wave runs first. Every index equals the plain model's."""
from __future__ import annotations

import re
import shutil
import struct
import subprocess
from pathlib import Path

import numpy as np
import pytest

from test_gpu_evict import model, random_weights

HERE = Path(__file__).resolve().parent
KERNELS = HERE.parent / "kv-compact_amd" / "csrc" / "kvc_evict.hip"
CLANG = "/opt/rocm/llvm/bin/clang++"


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    if not shutil.which(CLANG):
        pytest.skip("clang++ not available")
    d = tmp_path_factory.mktemp("pick")
    m = re.search(r"^constexpr int kPick.*?(?=^struct TakeArgs)", KERNELS.read_text(), re.S | re.M)
    assert m, "k_pick not found"
    (d / "pick.inc").write_text(m.group(0))
    b = subprocess.run([CLANG, "-std=c++17", "-O1", "-g", "-w", "-ffp-contract=off", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                        f"-I{d}", str(HERE / "waves" / "pick.cpp"), "-o", str(d / "pick")], capture_output=True, text=True, timeout=300)
    assert b.returncode == 0, b.stderr[-3000:]
    return d / "pick"


def run(exe, w, lens, seqs, start, keep, recent, first, most=False, shared=False, own=False, n_idx=None):
    L, n_seqs, H, room = w.shape
    if n_idx is None:
        n_idx = model(w, lens, seqs, start, keep, recent, most, shared, 1 << 40, max(lens), room)[1][-1]
    lists, cu, granted, status = model(w, lens, seqs, start, keep, recent, most, shared, n_idx, max(lens), room)
    n, groups = len(seqs), len(lists)
    head = struct.pack("<12i", own, first, L, n_seqs, H, room, n, n_idx, recent, most, groups, max(lens))
    r = subprocess.run([str(exe)], input=head + b"".join(np.int32(x).tobytes() for x in (lens, seqs, start, keep)) + w.tobytes(),
                       capture_output=True, timeout=300)
    assert r.returncode == 0, r.stderr.decode()[-3000:]
    out = np.frombuffer(r.stdout, np.int32)
    assert out[:3 * n + 1].tolist() == cu + granted + status
    got = out[3 * n + 1:].reshape(groups, n_idx)
    want = np.full(got.shape, -7)
    for g, per in enumerate(lists):
        for i, x in enumerate(per):
            want[g, cu[i]:cu[i + 1]] = x
    assert np.array_equal(got, want), np.argwhere(got != want)[:5].tolist()


# (a threshold of 1 has its place of the histogram cleared by wave 7, one of 0 by wave 0)
@pytest.mark.parametrize("first", [0, 7, 15, -1])
@pytest.mark.parametrize("own", [False, True])
def test_keys_near_the_threshold_in_lds(exe, first, own):
    rng = np.random.default_rng(1)
    w = (1 + 0.2 * rng.random((1, 1, 1, 2320))).astype(np.float32)
    run(exe, w, [2311], [0], [3], [700], 20, first, own=own)


@pytest.mark.parametrize("first", [0, 7, 15, -1])
def test_more_keys_than_lds_holds(exe, first):
    rng = np.random.default_rng(2)
    w = np.ones((1, 1, 1, 6000), np.float32)
    w[..., ::3] = 1 + 0.1 * rng.random((1, 1, 1, 2000))
    run(exe, w, [5990], [0], [0], [1500], 5, first)   # between the two kinds
    run(exe, w, [5990], [0], [0], [4000], 5, first)   # among equal ones
    run(exe, 0 * w, [5990], [0], [0], [4000], 5, first)


@pytest.mark.parametrize("shared,most", [(False, False), (True, False), (True, True)])
def test_requests_of_a_call(exe, shared, most):
    rng = np.random.default_rng(3)
    w = random_weights(rng, 2, 4, 2, 320)
    run(exe, w, [300, 0, 65, 17], [2, 0, 0, 9, 3], [1, 4, 0, 0, 0], [30, 150, 5, 3, 20], 7, 7, most, shared)
    run(exe, w, [300, 0, 65, 17], [2, 0, 3], [1, 4, 0], [30, 150, 5], 7, 7, most, shared, n_idx=60)


def test_more_requests_than_a_wave_has_lanes(exe):
    rng = np.random.default_rng(4)
    w = random_weights(rng, 1, 70, 1, 16)
    lens = rng.integers(0, 17, 70)
    run(exe, w, lens.tolist(), rng.permutation(70).tolist(), [0] * 70, rng.integers(0, 9, 70).tolist(), 2, 7)
