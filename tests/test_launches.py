"""The host side of the cache's calls under the undefined-behaviour sanitizer (tests/launches), with a runtime that records
launches: addresses far into large caches, and launches for every size that arguments can announce."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
CSRC = HERE.parent / "kv-compact_amd" / "csrc"
HIPCC = "/opt/rocm/bin/hipcc"
FLAGS = ["--offload-arch=gfx950", "--offload-host-only", "-O1", "-g", "-w", "-std=c++17", "-fPIC", "-ffp-contract=off",
         "-Xarch_host", "-fsanitize=undefined", "-Xarch_host", "-fno-sanitize-recover=undefined"]


def test_launches(tmp_path):
    if not shutil.which(HIPCC):
        pytest.skip("hipcc not available")
    sources = [CSRC / x for x in ("kvc_cache.hip", "kvc_attn.hip", "kvc_window.hip", "kvc_weigh.hip", "kvc_evict.hip")]
    objects = []
    for s in sources + [HERE / "launches" / "launches.cpp"]:
        objects.append(str(tmp_path / (s.stem + ".o")))
        b = subprocess.run([HIPCC, *FLAGS, "-x", "hip", "-c", str(s), "-o", objects[-1]], capture_output=True, text=True, timeout=300)
        assert b.returncode == 0, b.stderr[-2000:]
    # (no runtime and no device code: what is not recorded is not called)
    b = subprocess.run(["/opt/rocm/llvm/bin/clang++", "-fsanitize=undefined", "-Wl,--unresolved-symbols=ignore-all", *objects,
                        "-o", str(tmp_path / "launches")], capture_output=True, text=True, timeout=300)
    assert b.returncode == 0, b.stderr[-2000:]
    r = subprocess.run([str(tmp_path / "launches")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-3000:]
    assert int(r.stdout.split()[0]) > 100000, r.stdout
