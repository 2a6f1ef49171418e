"""The paged-serving ops' CPU references (csrc/core/paged_ref.cpp) on exactly sized
buffers under AddressSanitizer + UndefinedBehaviorSanitizer
(tests/native/test_paged.cpp), host code only."""
from __future__ import annotations

import os
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_paged_references_asan_ubsan(tmp_path):
    exe = tmp_path / "test_paged"
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer", "-fsanitize=address,undefined",
                        "-fno-sanitize-recover=undefined", f"-I{ROOT / 'csrc' / 'include'}",
                        str(ROOT / "csrc" / "core" / "paged_ref.cpp"), str(ROOT / "tests" / "native" / "test_paged.cpp"),
                        "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1")
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "ALL NATIVE TESTS PASSED" in r.stderr, r.stderr[-6000:]
