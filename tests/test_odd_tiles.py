"""Under a window, the search for values that are not finite goes through tiles of keys that some row sees, and through no
others, however long the sequence between its first cells and the window (the kernels' own code, on the CPU)."""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

HERE = Path(__file__).resolve().parent
KERNELS = HERE.parent / "kv-compact_amd" / "csrc" / "kvc_attn_kernels.h"
CLANG = "/opt/rocm/llvm/bin/clang++"


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    if not shutil.which(CLANG):
        pytest.skip("clang++ not available")
    d, text = tmp_path_factory.mktemp("odd"), ""
    for begin, end in (("// Where rows of K or V stand", "namespace {"), ("typedef float f4", "// Values of V that are not finite")):
        m = re.search(rf"^{begin}.*?(?=^{end})", KERNELS.read_text(), re.S | re.M)
        assert m, f"{begin} not found"
        text += m.group(0)
    text = re.sub(r"asm volatile\(.*?\);", ";", text, flags=re.S).replace("__attribute__((address_space(4)))", "")
    (d / "odd_tiles.inc").write_text(text)
    b = subprocess.run([CLANG, "-std=c++17", "-O1", "-g", "-w", "-mf16c", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                        f"-I{d}", str(HERE / "waves" / "odd_tiles.cpp"), "-o", str(d / "odd_tiles")],
                       capture_output=True, text=True, timeout=300)
    assert b.returncode == 0, b.stderr[-3000:]
    return d / "odd_tiles"


def test_only_tiles_that_some_row_sees(exe):
    rng = np.random.default_rng(0)
    cases = []
    for _ in range(400):
        cells = int(2 ** rng.uniform(5, 20))
        new = int(rng.integers(1, min(cells, 40) + 1))
        first, last = int(rng.choice([0, 4, 33, 100, 3000])), int(2 ** rng.uniform(0, 14))
        lo, hi = sorted(rng.integers(0, new, 2).tolist())
        tiles = -(-(cells - new + hi + 1) // 32)
        near, to = -(-first // 32), max(0, cells - new + lo + 1 - last) // 32
        seen = [t for t in range(tiles) if t < near or t >= to]
        at = int(rng.integers(0, len(seen))) if rng.random() < 0.5 else 0
        end = int(rng.integers(at + 1, len(seen) + 1))
        cases.append((first, last, cells, new, lo, hi, at, end, int(rng.integers(0, 1 << 20)) if rng.random() < 0.5 else 0, set(seen)))
    r = subprocess.run([str(exe)], input=np.int32([c[:9] for c in cases]).tobytes(), capture_output=True, timeout=60)
    assert r.returncode == 0, r.stderr.decode()[-2000:]
    out, i = np.frombuffer(r.stdout, np.int32).tolist(), 0
    for c in cases:
        marked, n = out[i], out[i + 1]
        pairs = [(out[i + 2 + 2 * j], out[i + 3 + 2 * j]) for j in range(n)]
        i += 2 + 2 * n
        gone = sum(e - b for b, e in pairs)
        stretch = 1 << max(0, (c[7] - c[6] - 1).bit_length() - 6)
        assert gone <= 32 * stretch, (c[:9], pairs)
        assert any(b <= 32 * marked and min(32 * marked + 32, c[2]) <= e for b, e in pairs), (c[:9], marked, pairs)
        assert all(t in c[9] for b, e in pairs for t in range(b // 32, -(-e // 32))), (c[:9], pairs)
    assert i == len(out)
